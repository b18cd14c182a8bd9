// Decode attention over pages of 8-bit keys and values (cache8.cuh): one query token per request.
//
// The split of the work is attention_decode_tma.cu's (64-key tiles brought by the copy engine into a ring, four warps with 16 keys of
// every tile each, the token's keys split over `splits` blocks and merged by decode_combine), and a warp's 16 keys are just one
// block of tokens with one scale.  Half the bytes come from memory, so what a warp does for a key has to take half the time:
//   * the 16 keys are the M side of mma.sync m16n8k16 and up to eight heads its N side (two such groups where a key/value head has
//     more query heads): scores K Q^T, then outputs V^T P^T with 16 elements of the head as M.  Heads as M fill seven of sixteen rows
//     in a group of seven; this way takes half the products, accumulators and exponentials.  Probabilities change sides by movmatrix.
//   * e4m3 numbers become float16 in one instruction for two (exact), and float16 is what is multiplied, not bfloat16: queries
//     are brought to 2^13 .. 2^14 per head by a power of two, which keeps all their bits.
//   * keys are read from shared memory 16 bytes at a time as they lie; which of the head's elements stand at which place of a
//     product's k index is free as long as the queries agree, and so is the order of a tile's keys.
//   * values are transposed in pairs of bytes by ldmatrix; one byte permute then gives the even and the odd column's pairs, which
//     are the two halves of a product's 16 rows.
//   * a block's scale of the keys goes into the exponent's factor.  Its values are weighed by probabilities that are relative to
//     the block's own largest one, times 2^7, in float16: eleven bits down to 2^-21 of that one (three more than in bfloat16) and off by
//     2^-32 of it at most below.  The block's sums join the warp's in float32, times the scale of its values and what its largest
//     probability is of the warp's, so that neither a weight nor a scale far from other blocks' costs any block its bits: with
//     both in the float16 numbers, relative to the largest scale the warp had met, a block of 2^-16 of that scale lost bits and one of
//     2^-25 was 0, whatever its weight.
// Values of keys that the query does not see are zeroed: what stands behind a request's last token in its page may be anything.
//
// With FRESH the kernel starts from the q/k/v product, which qkv_rope_store8 followed by it would do in two launches: it adds up the
// product's parts and the bias, rotates q (into shared memory) and the token's key, and the warp whose 16 keys are the token's own block
// rounds key and value, with the block's scale as cache8.cu says, puts them into the tile once it has landed (and rounds the block's
// earlier rows again there and in the page, where its scale grows), and writes page and scale.  No other block of the grid reads that
// block of tokens.  With `early` only what the product wrote is waited for: pages, tables and positions were written before the
// launch right ahead started, and the old keys are on their way while the product ends.
//
// Every wait on an mbarrier is bounded (tma.cuh); on giving up the block flags *status = 5.
#include "cache8.cuh"
#include "mma.cuh"
#include "tma.cuh"

namespace air {

constexpr int D8_CONSUMERS = 4;
constexpr int D8_THREADS = (D8_CONSUMERS + 1) * 32;
constexpr int D8_TILE = 64;     // keys per stage

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with nothing to add to.
__device__ __forceinline__ void mma_f16_16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// a += x f.x, b += y f.y, in one instruction.
__device__ __forceinline__ void add_two(float& a, float& b, float x, float y, float2 f) {
    asm("{\n\t.reg .b64 s, v, f;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 f, {%4, %5};\n\t"
        "fma.rn.f32x2 s, v, f, s;\n\tmov.b64 {%0, %1}, s;\n\t}"
        : "+f"(a), "+f"(b) : "f"(x), "f"(y), "f"(f.x), "f"(f.y));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
// An 8 x 8 matrix of 16-bit elements, two of a row to a lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// 2^x by the special-function unit (2^-22 off; what falls below 2^-126 becomes 0, which a rounding to float16 does anyway).
__device__ __forceinline__ float exp2_quick(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void tma_load_3d_hint(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
__device__ __forceinline__ float exp2_int(int e) { return e < -126 ? 0.f : __uint_as_float((uint32_t)(min(e, 127) + 127) << 23); }

// A [64][D] tile of bytes with the swizzle of its row length (128 or 64 bytes): the address of a 16-byte chunk.
template <int D>
__device__ __forceinline__ uint32_t chunk8(uint32_t tile, int row, int chunk) {
    return D == 128 ? tile + row * 128 + ((chunk ^ (row & 7)) << 4) : tile + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}
// Which of eight keys stands at place i of a product's eight: in rows of 128 bytes two neighbouring places are four rows apart, so
// that the eight lanes that read at once (two keys, four chunks each) meet all banks.
template <int D>
__device__ __forceinline__ int key_at(int i) { return D == 128 ? (i >> 1) | ((i & 1) << 2) : i; }

// The largest finite |number| of a row that a warp holds, as bits.
template <int D>
__device__ __forceinline__ uint32_t top_of_row(const Row8<D>& r) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < Row8<D>::N; ++e) {
        const uint32_t a = __float_as_uint(r.a[e]) & 0x7fffffffu, b = __float_as_uint(r.b[e]) & 0x7fffffffu;
        if (a < 0x7f800000u) top = max(top, a);
        if (b < 0x7f800000u) top = max(top, b);
    }
    return __reduce_max_sync(0xffffffffu, top);
}

// A warp puts the row of position pos into its tile in shared memory and into the page (null: not there), the head's rows of which
// begin at `page`; `need` is the scale that the row asks for, `kept` the block's so far (0: the row is its first).  Returns the
// block's scale, for which its earlier rows have been rounded again where it has grown.
template <int D>
__device__ __forceinline__ float put_row(const Row8<D>& r, float need, float kept, uint32_t tile, uint8_t* page, int pos, int P, int lane) {
    constexpr int N = Row8<D>::N;
    const float scale = fmaxf(kept, need), down = 1.f / scale;      // (powers of two: exact)
    const int row = pos % D8_TILE, first = pos % BLOCK8, in_page = pos % P;
    auto scaled = [&](float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u ? x * down : __uint_as_float(0x7fc00000u); };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int e = lane * N + half * (D / 2);
        const float* v = half ? r.b : r.a;
        const uint32_t code = to_e4m3x2(scaled(v[0]), N == 2 ? scaled(v[N - 1]) : 0.f), at = chunk8<D>(tile, row, e >> 4) + (e & 15);
        if constexpr (N == 2) {
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)code) : "memory");
            if (page) *reinterpret_cast<uint16_t*>(page + (size_t)in_page * D + e) = (uint16_t)code;
        } else {
            asm volatile("st.shared.u8 [%0], %1;" ::"r"(at), "r"(code & 0xffu) : "memory");
            if (page) page[(size_t)in_page * D + e] = (uint8_t)code;
        }
    }
    if (scale > kept && first > 0) {
        const float less = kept * down;
        constexpr int E = D / 32;               // bytes of a row to a lane
        for (int i = 0; i < first; ++i) {
            const uint32_t at = chunk8<D>(tile, row - first + i, (lane * E) >> 4) + ((lane * E) & 15);
#pragma unroll
            for (int c = 0; c < E / 2; ++c) {
                uint16_t code;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(code) : "r"(at + 2 * c) : "memory");
                const float2 x = e4m3x2_to_float2(code);
                code = to_e4m3x2(x.x * less, x.y * less);
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + 2 * c), "h"(code) : "memory");
                if (page) *reinterpret_cast<uint16_t*>(page + (size_t)(in_page - first + i) * D + lane * E + 2 * c) = code;
            }
        }
    }
    return scale;
}

// The token's new q, k and v as the product left them (FRESH).
struct Fresh8 {
    const float* qkv;        // [parts][T][(H + 2 K) D]
    int parts;
    size_t part_stride;
    const float *bias, *table;
    uint8_t* cache;          // where key and value are written (null: another run's layer has written them)
    float* scales;
    int early;
};

// GROUPS: of eight heads that a block takes, 1 or 2.  FEW: the grid is no larger than two blocks an SM, which then have six stages each
// and registers for as many; of a larger one four share an SM, with three.  us with six stages and with three: one of 512 7.4 / 7.8, of
// 2,048 8.4 / 9.5; 16 of 512 9.2 / 11.3, of 2,048 13.9 / 19.0; 64 of 100 to 8,192 75 / 64, 256 of 200 28 / 20 (from there on it is
// the number of warps that counts: some 350 instructions for a warp's 16 keys, most of them behind one another).
template <int D, int GROUPS, bool FRESH, bool FEW>
__global__ void __launch_bounds__(D8_THREADS, GROUPS == 1 && !FEW ? 4 : 2)
decode_attention8_kernel(const __grid_constant__ CUtensorMap map_cache, const Fresh8 fresh, const float* __restrict__ scales, const __nv_bfloat16* __restrict__ q,
                         const int* __restrict__ block_table, int max_blocks, const int* __restrict__ token_seq,
                         const int* __restrict__ positions, __nv_bfloat16* __restrict__ out, float* __restrict__ part_o,
                         float* __restrict__ part_ml, int H, int K, int P, int window, float scale_log2, int least, int* status) {
    // least: tiles of a split at least, so that a short context is one block's work and needs no merge
    constexpr int TILE_BYTES = D8_TILE * D, STAGE_BYTES = 2 * TILE_BYTES, STAGES = FEW ? 6 : 3;
    constexpr int PIECES = D / 64;              // chunks of a key's row that a lane reads (16 bytes, four steps of k)
    constexpr int CH = D / 16;                  // 16-byte chunks of a row: 16 rows of the outputs' product each
    constexpr int ROWS = 8 * GROUPS;            // heads of a block
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + STAGES * STAGE_BYTES);
    uint64_t* empty = full + STAGES;
    volatile int* abort_flag = (volatile int*)(empty + STAGES);
    float* sm_o = (float*)smem;                              // after the walk: [warps][ROWS][D]
    float* sm_m = sm_o + D8_CONSUMERS * ROWS * D;            // [warps][ROWS]
    float* sm_l = sm_m + D8_CONSUMERS * ROWS;

    uint8_t* sm_q = (uint8_t*)(empty + STAGES) + 16;      // FRESH: [ROWS][D] bfloat16

    pdl_trigger();
    if (!FRESH || !fresh.early) pdl_wait();
    trace_point(TR_ATT_DECODE);
    // (a block without keys does no more than this)
    const int t = blockIdx.z;
    const int slot = token_seq[t], pos = positions[t];
    if (slot < 0 || pos < 0 || pos / P >= max_blocks) {      // (the last: a position that the table has no place for)
        if (FRESH && fresh.early) pdl_wait();                // (a grid of none but such tokens must not be over before the product)
        if (slot >= 0 && pos >= 0 && threadIdx.x == 0 && status) atomicExch(status, 2);
        return;
    }
    const int lo = window > 0 ? max(0, pos - window + 1) : 0;
    const int split = blockIdx.x, splits = gridDim.x;
    const int tile0 = lo / D8_TILE, tile1 = pos / D8_TILE + 1;
    const int per = max(least, (tile1 - tile0 + splits - 1) / splits);
    const bool alone = tile1 - tile0 <= per;                 // all of the token's keys are one split's
    const int begin = tile0 + split * per, end = min(tile1, begin + per);
    const int n_tiles = end - begin;
    if (n_tiles <= 0) return;                                // (the merge does not read this split's numbers)
    const int* bt = block_table + (size_t)slot * max_blocks;
    const int G = H / K, head_blocks = (G + ROWS - 1) / ROWS;
    const int kvh = blockIdx.y / head_blocks, hb = blockIdx.y % head_blocks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], D8_CONSUMERS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    uint64_t kv_policy;         // (keys and values pass through L2 once)
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(kv_policy));

    const int g = lane >> 2, tq = lane & 3;
    // o[x][n]: of group x's heads 2 tq and 2 tq + 1, elements 16 n + 2 g (first two) and 16 n + 2 g + 1; m, l: of the same two heads
    float o[GROUPS][CH][4], m[GROUPS][2], l[GROUPS][2];
#pragma unroll
    for (int x = 0; x < GROUPS; ++x) {
#pragma unroll
        for (int n = 0; n < CH; ++n) o[x][n][0] = o[x][n][1] = o[x][n][2] = o[x][n][3] = 0.f;
        m[x][0] = m[x][1] = -INFINITY;
        l[x][0] = l[x][1] = 0.f;
    }

    if (warp == D8_CONSUMERS) {
        // ------------------------------------------------------------ copies
        // Lane i looks up the pages of 32 boxes at once (a page at a time is a round trip to L2 ahead of every tile), and keys and values of
        // whole tiles come in one copy: asking for a copy costs the thread some 200 cycles, and a tile in two of them took longer to ask
        // for than to read.
        const int box_rows = P < D8_TILE ? P : D8_TILE, boxes = D8_TILE / box_rows;
        int page = 0, row = 0;
        for (int it = 0; it < n_tiles; ++it) {
            const int stage = it % STAGES, kbase = (begin + it) * D8_TILE, box0 = it * boxes & 31;
            if (box0 == 0) {
                const int first = kbase + lane * box_rows;
                page = first <= pos && first + box_rows - 1 >= lo ? bt[first / P] : 0;
                row = kvh * P + first % P;
            }
            if (it >= STAGES && !__all_sync(0xffffffffu, mbar_wait(&empty[stage], ((it / STAGES) - 1) & 1, abort_flag))) break;
            int valid = 0;
            for (int b = 0; b < boxes; ++b) {
                const int first = kbase + b * box_rows;
                valid += (first <= pos && first + box_rows - 1 >= lo) ? 1 : 0;
            }
            if (lane == 0) mbar_expect_tx(&full[stage], (uint32_t)(valid * box_rows * D * 2));
            uint8_t* dst = smem + stage * STAGE_BYTES;
            for (int b = 0; b < boxes; ++b) {
                const int first = kbase + b * box_rows, of = __shfl_sync(0xffffffffu, page, box0 + b), at = __shfl_sync(0xffffffffu, row, box0 + b);
                if (!(first <= pos && first + box_rows - 1 >= lo) || lane != 0) continue;
                tma_load_3d_hint(dst + b * box_rows * D, &map_cache, 0, at, 2 * of, &full[stage], kv_policy);
                if (boxes > 1) tma_load_3d_hint(dst + TILE_BYTES + b * box_rows * D, &map_cache, 0, at, 2 * of + 1, &full[stage], kv_policy);
            }
        }
    } else {
        // ------------------------------------------------------------ 16 keys of every tile each
        // lane i: the scales of the warp's block of tile it + i (the first ones asked for ahead of the queries)
        float scale_k = 0.f, scale_v = 0.f;
        auto ask_scales = [&](int it) {
            const int first = (begin + it + lane) * D8_TILE + 16 * warp;
            scale_k = scale_v = 0.f;
            if (it + lane < n_tiles && first <= pos && first + 15 >= lo) {
                const int page = bt[first / P];
                if (page >= 0) {
                    const size_t at = ((size_t)page * 2 * K + kvh) * (P / BLOCK8) + first % P / BLOCK8;
                    scale_k = scales[at];
                    scale_v = scales[at + (size_t)K * (P / BLOCK8)];
                }
            }
        };
        ask_scales(0);
        // FRESH: the token's key and value are the work of the warp whose block of its tile they fall into
        const int own = pos % D8_TILE / BLOCK8;
        const bool mine = FRESH && fresh.cache && warp == own && end == tile1;
        Row8<D> new_k, new_v;
        float new_sk = 0.f, new_sv = 0.f;
        if constexpr (FRESH) {
            if (fresh.early) pdl_wait();
            // the warp's query heads, every fourth, and the key and value (asked for by all warps: a warp's rows are on their way at once)
            constexpr int MINE = ROWS / D8_CONSUMERS, ALL = MINE + 2;
            const size_t token = (size_t)t * (H + 2 * K) * D;
            size_t from[ALL];
            int head[ALL], at[ALL];
#pragma unroll
            for (int i = 0; i < ALL; ++i) {
                head[i] = (i < MINE ? kvh * G + min(warp + D8_CONSUMERS * i, G - 1) : i == MINE ? H + kvh : H + K + kvh) * D;
                from[i] = token + head[i];
                at[i] = pos;
            }
            Row8<D> v[ALL];
            product_rows<D, ALL, GROUPS == 1 ? 3 : 1>(fresh.qkv, from, fresh.parts, fresh.part_stride, fresh.bias, head, lane, v);
            new_v = v[MINE + 1];
            turn_rows<D, ALL>(fresh.table, at, lane, v);
            new_k = v[MINE];
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int r = warp + D8_CONSUMERS * i;
                if (r >= G) break;
                __nv_bfloat16* to = (__nv_bfloat16*)sm_q + r * D + lane * Row8<D>::N;
#pragma unroll
                for (int e = 0; e < Row8<D>::N; ++e) {
                    to[e] = __float2bfloat16_rn(v[i].a[e]);
                    to[D / 2 + e] = __float2bfloat16_rn(v[i].b[e]);
                }
            }
            if (mine) {
                new_sk = scale8(top_of_row<D>(new_k));
                new_sv = scale8(top_of_row<D>(new_v));
            }
            asm volatile("bar.sync 1, %0;" ::"n"(D8_CONSUMERS * 32) : "memory");
        }
        // The queries of head g of each group: the lane holds the 16 elements of chunk tq (and tq + 4), four to a step of k.
        uint32_t qb[GROUPS][PIECES][4][2];
        float factor[GROUPS][2];                      // of heads 2 tq, 2 tq + 1
#pragma unroll
        for (int x = 0; x < GROUPS; ++x) {
            const int r = hb * ROWS + 8 * x + g;
            const uint4* src = FRESH ? reinterpret_cast<const uint4*>(sm_q + (8 * x + g) * D * 2)
                                     : reinterpret_cast<const uint4*>(q + ((size_t)t * H + kvh * G + r) * D);
            uint4 raw[PIECES][2];
            float top = 0.f;
#pragma unroll
            for (int hf = 0; hf < PIECES; ++hf)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    raw[hf][i] = r < G ? (FRESH ? src[2 * (tq + 4 * hf) + i] : __ldg(src + 2 * (tq + 4 * hf) + i)) : make_uint4(0u, 0u, 0u, 0u);
                    const uint32_t w[4] = {raw[hf][i].x, raw[hf][i].y, raw[hf][i].z, raw[hf][i].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // a head of zeros, and one of numbers below 2^-87, stays where it is put
            const int e = max(-100, (int)(__float_as_uint(top) >> 23) - 127 - 13);
            const float down = exp2_int(-e), up = scale_log2 * exp2_int(e);
            factor[x][0] = __shfl_sync(0xffffffffu, up, 8 * tq);
            factor[x][1] = __shfl_sync(0xffffffffu, up, 8 * tq + 4);
#pragma unroll
            for (int hf = 0; hf < PIECES; ++hf)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const uint4 v = raw[hf][s >> 1];
                    const uint32_t lo2 = s & 1 ? v.z : v.x, hi2 = s & 1 ? v.w : v.y;
                    qb[x][hf][s][0] = pack_f16(__uint_as_float(lo2 << 16) * down, __uint_as_float(lo2 & 0xffff0000u) * down);
                    qb[x][hf][s][1] = pack_f16(__uint_as_float(hi2 << 16) * down, __uint_as_float(hi2 & 0xffff0000u) * down);
                }
        }
        const int mat = lane >> 3, mrow = lane & 7;   // ldmatrix: which 8x8 matrix this lane addresses, which row
        bool alive = true;
        for (int it = 0; it < n_tiles; ++it) {
            if ((it & 31) == 0 && it > 0) ask_scales(it);
            float sk = __shfl_sync(0xffffffffu, scale_k, it & 31), sv = __shfl_sync(0xffffffffu, scale_v, it & 31);
            const int stage = it % STAGES;
            // (a warp whose wait ran out goes on without work, so that it still meets the others at the barrier below)
            if (alive) alive = __all_sync(0xffffffffu, mbar_wait(&full[stage], (it / STAGES) & 1, abort_flag));
            if (!alive) continue;
            const int kbase = (begin + it) * D8_TILE + 16 * warp;     // this warp's 16 keys
            if (kbase <= pos && kbase + 15 >= lo) {
                const uint32_t kt = smem_u32(smem + stage * STAGE_BYTES), vt = kt + TILE_BYTES;
                if (FRESH && mine && begin + it == tile1 - 1) {
                    const int page = bt[pos / P], first = pos % BLOCK8;
                    const size_t line = ((size_t)max(page, 0) * 2 * K + kvh) * P;            // the head's first key in the page; K P further, its first value
                    if (page < 0 && lane == 0 && status) atomicExch(status, 2);
                    sk = put_row<D>(new_k, new_sk, first > 0 ? sk : 0.f, kt, page < 0 ? nullptr : fresh.cache + line * D, pos, P, lane);
                    sv = put_row<D>(new_v, new_sv, first > 0 ? sv : 0.f, vt, page < 0 ? nullptr : fresh.cache + (line + (size_t)K * P) * D, pos, P, lane);
                    if (page >= 0 && lane == 0) {
                        float* sp = fresh.scales + line / BLOCK8 + pos % P / BLOCK8;
                        sp[0] = sk;
                        sp[(size_t)K * (P / BLOCK8)] = sv;
                    }
                    __syncwarp();
                }
                // scores: rows are keys (place g of the warp's first eight and of its second), columns heads 2 tq and 2 tq + 1
                // (two sums each, which do not wait for one another)
                float s[GROUPS][4] = {}, also[GROUPS][4] = {};
#pragma unroll
                for (int hf = 0; hf < PIECES; ++hf) {
                    uint32_t w[2][4];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[j][0]), "=r"(w[j][1]), "=r"(w[j][2]), "=r"(w[j][3])
                                     : "r"(chunk8<D>(kt, 16 * warp + 8 * j + key_at<D>(g), tq + 4 * hf)));
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)w[0][k]), a1 = e4m3x2_to_f16x2((uint16_t)w[1][k]);
                        const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)(w[0][k] >> 16)), a3 = e4m3x2_to_f16x2((uint16_t)(w[1][k] >> 16));
#pragma unroll
                        for (int x = 0; x < GROUPS; ++x) mma_f16_16816(k & 1 ? also[x] : s[x], a0, a1, a2, a3, qb[x][hf][k][0], qb[x][hf][k][1]);
                    }
                }
                const bool whole = kbase >= lo && kbase + 15 <= pos;
                auto seen = [&](int place) { return kbase + place >= lo && kbase + place <= pos; };
                float top_here[GROUPS][2];      // the block's largest scores
                bool move = false;
#pragma unroll
                for (int x = 0; x < GROUPS; ++x) {
                    const float f0 = factor[x][0] * sk, f1 = factor[x][1] * sk;
                    s[x][0] = (s[x][0] + also[x][0]) * f0, s[x][1] = (s[x][1] + also[x][1]) * f1;
                    s[x][2] = (s[x][2] + also[x][2]) * f0, s[x][3] = (s[x][3] + also[x][3]) * f1;
                    if (!whole) {
                        if (!seen(key_at<D>(g))) s[x][0] = s[x][1] = -INFINITY;
                        if (!seen(8 + key_at<D>(g))) s[x][2] = s[x][3] = -INFINITY;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float tm = fmaxf(s[x][h], s[x][2 + h]);
                        tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 4));
                        tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 8));
                        tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, 16));
                        // (at least one key is visible; a block whose scores have all run to -infinity weighs nothing)
                        top_here[x][h] = fmaxf(tm, -3e38f);
                        move |= top_here[x][h] > m[x][h];
                    }
                }
                if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                    for (int x = 0; x < GROUPS; ++x)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float top = fmaxf(m[x][h], top_here[x][h]), c = exp2_quick(m[x][h] - top);
                            m[x][h] = top;
                            l[x][h] *= c;
#pragma unroll
                            for (int n = 0; n < CH; ++n) o[x][n][h] *= c, o[x][n][2 + h] *= c;
                        }
                }
                uint32_t pb[GROUPS][2];
                float2 unit[GROUPS];      // what the block's sums are of the warp's
#pragma unroll
                for (int x = 0; x < GROUPS; ++x) {
                    // (7: where scores are so large that the difference is rounded, it is 8 at most)
                    const float from0 = top_here[x][0] - 7.f, from1 = top_here[x][1] - 7.f;
                    const float of0 = exp2_quick(from0 - m[x][0]), of1 = exp2_quick(from1 - m[x][1]);
                    unit[x] = make_float2(of0 * sv, of1 * sv);
                    float p[2][2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        p[j][0] = exp2_quick(s[x][2 * j] - from0);
                        p[j][1] = exp2_quick(s[x][2 * j + 1] - from1);
                        pb[x][j] = transposed(pack_f16(p[j][0], p[j][1]));
                    }
                    l[x][0] = fmaf(p[0][0] + p[1][0], of0, l[x][0]);
                    l[x][1] = fmaf(p[0][1] + p[1][1], of1, l[x][1]);
                }
                uint32_t live[2] = {0xffffffffu, 0xffffffffu};
                if (!whole)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        live[j] = (seen(8 * j + key_at<D>(2 * tq)) ? 0x0000ffffu : 0u) | (seen(8 * j + key_at<D>(2 * tq + 1)) ? 0xffff0000u : 0u);
#pragma unroll
                for (int n = 0; n < CH; n += 2) {
                    // matrices: (keys 0-7, chunk n), (keys 8-15, chunk n), (keys 0-7, chunk n + 1), (keys 8-15, chunk n + 1), a pair of
                    // neighbouring columns to an element
                    uint32_t b[4];
                    ldmatrix_x4_trans(b, chunk8<D>(vt, 16 * warp + 8 * (mat & 1) + key_at<D>(mrow), n + (mat >> 1)));
                    if (!whole) {
                        b[0] &= live[0];
                        b[1] &= live[1];
                        b[2] &= live[0];
                        b[3] &= live[1];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) b[i] = __byte_perm(b[i], 0, 0x3120);      // the even column's two keys, the odd one's
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)b[2 * i]), a1 = e4m3x2_to_f16x2((uint16_t)(b[2 * i] >> 16));
                        const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)b[2 * i + 1]), a3 = e4m3x2_to_f16x2((uint16_t)(b[2 * i + 1] >> 16));
#pragma unroll
                        for (int x = 0; x < GROUPS; ++x) {
                            float here[4];
                            mma_f16_16816_first(here, a0, a1, a2, a3, pb[x][0], pb[x][1]);
                            add_two(o[x][n + i][0], o[x][n + i][1], here[0], here[1], unit[x]);
                            add_two(o[x][n + i][2], o[x][n + i][3], here[2], here[3], unit[x]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
        }
#pragma unroll
        for (int x = 0; x < GROUPS; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 4; i < 32; i *= 2) l[x][h] += __shfl_xor_sync(0xffffffffu, l[x][h], i);
    }

    // ---------------------------------------------------------------- merge the four warps
    __syncthreads();   // every tile has been consumed: the ring's memory is used again
    if (*abort_flag) {
        for (int i = 0; i < 32; ++i) __nanosleep(2000);   // copies on their way may still land
        if (threadIdx.x == 0 && status) atomicExch(status, 5);
        return;
    }
    if (warp < D8_CONSUMERS) {
#pragma unroll
        for (int x = 0; x < GROUPS; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = warp * ROWS + 8 * x + 2 * tq + h;
                if (g == 0) sm_m[row] = m[x][h], sm_l[row] = l[x][h];
#pragma unroll
                for (int n = 0; n < CH; ++n)
                    *reinterpret_cast<float2*>(sm_o + row * D + 16 * n + 2 * g) = make_float2(o[x][n][h], o[x][n][2 + h]);
            }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < min(ROWS, G - hb * ROWS) * D; idx += D8_THREADS) {
        const int r = idx / D, col = idx % D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < D8_CONSUMERS; ++w) mm = fmaxf(mm, sm_m[w * ROWS + r]);
        float acc = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < D8_CONSUMERS; ++w) {
            const float wgt = sm_m[w * ROWS + r] == -INFINITY ? 0.f : exp2f(sm_m[w * ROWS + r] - mm);
            acc += sm_o[(w * ROWS + r) * D + col] * wgt;
            ll += sm_l[w * ROWS + r] * wgt;
        }
        const int h = kvh * G + hb * ROWS + r;
        if (alone) {
            out[((size_t)t * H + h) * D + col] = __float2bfloat16_rn(acc / ll);
        } else {
            const size_t pi = ((size_t)t * H + h) * splits + split;
            part_o[pi * D + col] = acc;
            if (col == 0) {
                // (a split whose scores are all NaN has no largest one: the merge would pass it over)
                part_ml[pi * 2] = ll != ll ? 3e38f : mm;
                part_ml[pi * 2 + 1] = ll;
            }
        }
    }
}

template <int D, int GROUPS, bool FRESH, bool FEW>
static int launch_decode8_on(const CUtensorMap& map, const Fresh8& fresh, const float* scales, const void* q, const int* block_table, int max_blocks,
                          const int* token_seq, const int* positions, void* out, float* part_o, float* part_ml, int T, int H, int K, int P,
                          int window, float scale, int splits, int least, int* status, cudaStream_t stream) {
    constexpr int ROWS = 8 * GROUPS, STAGES = FEW ? 6 : 3;
    const size_t ring = (size_t)STAGES * 2 * D8_TILE * D + 2 * STAGES * 8 + 16 + (FRESH ? ROWS * D * 2 : 0);
    const size_t merge = (size_t)(D8_CONSUMERS * ROWS * D + 2 * D8_CONSUMERS * ROWS) * sizeof(float);
    const size_t smem = 1024 + (ring > merge ? ring : merge);
    auto kernel = decode_attention8_kernel<D, GROUPS, FRESH, FEW>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    return launch(kernel, dim3(splits, K * ((H / K + ROWS - 1) / ROWS), T), D8_THREADS, smem, stream, map, fresh, scales, (const __nv_bfloat16*)q, block_table,
                  max_blocks, token_seq, positions, (__nv_bfloat16*)out, part_o, part_ml, H, K, P, window, scale * 1.4426950408889634f, least, status);
}

template <int D, int GROUPS, bool FRESH>
static int launch_decode8(const CUtensorMap& map, const Fresh8& fresh, const float* scales, const void* q, const int* block_table, int max_blocks,
                          const int* token_seq, const int* positions, void* out, float* part_o, float* part_ml, int T, int H, int K, int P,
                          int window, float scale, int splits, int least, int* status, cudaStream_t stream) {
    const long long blocks = (long long)splits * T * K * ((H / K + 8 * GROUPS - 1) / (8 * GROUPS));
    return (blocks <= 2 * 148 ? launch_decode8_on<D, GROUPS, FRESH, true> : launch_decode8_on<D, GROUPS, FRESH, false>)(
        map, fresh, scales, q, block_table, max_blocks, token_seq, positions, out, part_o, part_ml, T, H, K, P, window, scale, splits, least, status, stream);
}

}  // namespace air

// The merge of the splits (attention_decode.cu).
extern "C" int air_decode_combine_least(const float* part_o, const float* part_ml, const int* token_seq, void* out, int T, int H, int D,
                                        int splits, const int* positions, int window, int early, int least, cudaStream_t stream);

namespace air {
static int decode_attention8(const Fresh8& fresh, const void* q, const void* cache, const float* scales, long long pages, const int* block_table,
                             int max_blocks, const int* token_seq, const int* positions, void* out, float* part_o, float* part_ml, int T, int H, int K,
                             int D, int P, int window, float scale, int splits, int least, int* status, cudaStream_t stream) {
    if (T <= 0) return T < 0 ? AIR_ERR_BAD_ARGUMENT : 0;
    if (H <= 0 || K <= 0 || H % K || P < BLOCK8 || P % BLOCK8 || (P < D8_TILE ? D8_TILE % P : P % D8_TILE) || splits < 1 || least < 1 || T > 65535 ||
        (long long)K * ((H / K + 7) / 8) > 65535 || window < 0 || (splits > 1 && (!part_o || !part_ml)) || (((uintptr_t)cache | (uintptr_t)q) & 15) ||
        (D != 64 && D != 128) || pages * 2 * K * P > 0x7fffffffll)
        return AIR_ERR_BAD_ARGUMENT;
    CUtensorMap map;
    int rc = rows8_map(&map, cache, pages, K * P, D, P < D8_TILE ? P : D8_TILE);
    if (rc) return rc;
    auto go = fresh.qkv ? (H / K <= 8 ? (D == 64 ? launch_decode8<64, 1, true> : launch_decode8<128, 1, true>)
                                      : (D == 64 ? launch_decode8<64, 2, true> : launch_decode8<128, 2, true>))
                        : (H / K <= 8 ? (D == 64 ? launch_decode8<64, 1, false> : launch_decode8<128, 1, false>)
                                      : (D == 64 ? launch_decode8<64, 2, false> : launch_decode8<128, 2, false>));
    rc = go(map, fresh, scales, q, block_table, max_blocks, token_seq, positions, out, part_o, part_ml, T, H, K, P, window, scale, splits, least, status,
            stream);
    if (rc || splits == 1) return rc;
    return air_decode_combine_least(part_o, part_ml, token_seq, out, T, H, D, splits, positions, window, 0, least, stream);
}
}  // namespace air

// q bfloat16 [T, H, D]; cache e4m3 and scales as in cache8.cuh, `pages` of them; the rest as air_decode_attention_tma
// (attention_decode_tma.cu).  Head size 64 or 128.  least: tiles of 64 keys that a split takes at least.
AIR_API int air_decode_attention8(const void* q, const void* cache, const float* scales, long long pages, const int* block_table, int max_blocks,
                                  const int* token_seq, const int* positions, void* out, float* part_o, float* part_ml, int T, int H, int K,
                                  int D, int P, int window, float scale, int splits, int least, int* status, cudaStream_t stream) {
    return air::decode_attention8(air::Fresh8{}, q, cache, scales, pages, block_table, max_blocks, token_seq, positions, out, part_o, part_ml, T, H, K, D,
                                  P, window, scale, splits, least, status, stream);
}

// The same from the q/k/v product instead of q, up to 16 query heads to a key/value head: qkv float32 [parts][T][(H + 2 K) D], bias
// float32 or null, table float32 [positions][D] (cos | sin).  write_kv 0: another run's layer has written keys and values.  early: pages,
// scales, tables and positions were written before the stream's last launch started.
AIR_API int air_decode_attention8_fresh(const float* qkv, int parts, const float* bias, const float* table, int write_kv, int early, void* cache,
                                        float* scales, long long pages, const int* block_table, int max_blocks, const int* token_seq,
                                        const int* positions, void* out, float* part_o, float* part_ml, int T, int H, int K, int D, int P, int window,
                                        float scale, int splits, int least, int* status, cudaStream_t stream) {
    if (!qkv || !table || parts < 1 || K < 1 || H / K > 16 || (((uintptr_t)qkv | (uintptr_t)bias | (uintptr_t)table) & 7)) return AIR_ERR_BAD_ARGUMENT;
    const air::Fresh8 fresh{qkv, parts, (size_t)T * (size_t)(H + 2 * K) * (size_t)D, bias, table, write_kv ? (uint8_t*)cache : nullptr, scales, early};
    return air::decode_attention8(fresh, nullptr, cache, scales, pages, block_table, max_blocks, token_seq, positions, out, part_o, part_ml, T, H, K, D, P,
                                  window, scale, splits, least, status, stream);
}

AIR_API int air_trace_set_attention_decode8(unsigned long long* buffer) { return air::set_trace_here(buffer); }
