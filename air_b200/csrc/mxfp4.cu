// Microscaled 4-bit floating point: rounding rows of numbers to it, reading them back, and products of two matrices held so.
//
// A block of 32 consecutive numbers of a row shares a scale 2^e and holds 32 e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives): x ~ q 2^e with e the smallest exponent (-127 at least) for which the block's largest number is at most 6 * 2^e, so
// that no number is cut off, and q = x / 2^e to the nearest, ties to even (e stays at 125, beyond which 6 * 2^e is no float32: larger
// numbers become 6 * 2^125).  A row may be held as the sum of several such numbers
// ("terms"): term t + 1 rounds what term t has left, which is exact in float32 (what is left of a number has no lower bits
// than the number or its rounded value has, and is smaller).  Each term leaves a sixth of the block's largest number at most.
// A block with a number that is not finite gets the scale NaN (byte 255): its products are NaN and not silently cut.
//
// packed [terms][rows][k / 2]: two numbers to a byte, the even one in the low half.
// scales [terms][row tiles][k tiles][32][16]: the bytes e + 127 in the tiles of 128 rows and 4 scales (128 numbers of k) that
// the tensor cores take: row r, scale j lies in tile (r / 128, j / 4) at byte (r % 32) * 16 + (r / 32 % 4) * 4 + j % 4.  The number
// of k tiles is even (a step of the product is 256 numbers of k); tiles past k hold zeros, rows past the last are not written.
#include "common.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace air {

// ------------------------------------------------------------------------------------------------ rounding
__device__ __forceinline__ float power_of_two(int e) {      // -127 <= e <= 127
    return __uint_as_float(e > -127 ? (uint32_t)(e + 127) << 23 : 0x00400000u);
}

// The byte of the scale of a block whose largest |number| has these bits: 6 = 1.5 * 2^2.
__device__ __forceinline__ int scale_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    return min(252, max(0, (int)(top >> 23) - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0)));
}

// Eight numbers of at most 6 to e2m1, the first in the lowest four bits.
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&y)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return r;
}

// And back: two bits of exponent and one of mantissa at a float32's place stand for the number times 2^-126 (0.5 is one of
// float32's own subnormal numbers there).
__device__ __forceinline__ void from_e2m1x8(uint32_t code, float (&y)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t c = code >> (4 * i);
        y[i] = __uint_as_float((c & 7u) << 22 | (c & 8u) << 28) * 8.507059173023462e37f;
    }
}

// Eight numbers of a row as they come, their largest magnitude's bits as a float32's, and they times a power of two.
template <typename T> struct Eight;
template <> struct Eight<__nv_bfloat16> {
    uint4 v;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ uint32_t top() const {
        const uint32_t m = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
        return max(m << 16, m & 0xffff0000u);
    }
    __device__ __forceinline__ void times(float f, float (&y)[8]) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[2 * i] = __uint_as_float(w[i] << 16) * f;
            y[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * f;
        }
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ uint32_t top() const {
        const float m[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) t = max(t, __float_as_uint(m[i]) & 0x7fffffffu);
        return t;
    }
    __device__ __forceinline__ void times(float f, float (&y)[8]) const {
        y[0] = a.x * f, y[1] = a.y * f, y[2] = a.z * f, y[3] = a.w * f;
        y[4] = b.x * f, y[5] = b.y * f, y[6] = b.z * f, y[7] = b.w * f;
    }
};

// Sixteen numbers from a boundary of 32 bytes, in copies of as many; they are not wanted again and leave L2 first.
__device__ __forceinline__ void load_32_bytes(const void* p, uint4& a, uint4& b) {
    asm volatile("ld.global.L2::evict_first.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
}
__device__ __forceinline__ void load_sixteen(const __nv_bfloat16* p, Eight<__nv_bfloat16> (&v)[2]) { load_32_bytes(p, v[0].v, v[1].v); }
__device__ __forceinline__ void load_sixteen(const float* p, Eight<float> (&v)[2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) load_32_bytes(p + 8 * h, reinterpret_cast<uint4&>(v[h].a), reinterpret_cast<uint4&>(v[h].b));
}

constexpr int MXQ_THREADS = 256;

// A warp takes 256 numbers of a row, a lane eight of them: four lanes are a block, sixteen the four scales of a tile's row.  For few
// rows, where the time is one round trip to memory and the launch.
// The successor is let off only behind the wait, so that what it reads ahead of its own wait (a product's weights) was written
// before this kernel started.
template <typename T>
__global__ void __launch_bounds__(MXQ_THREADS)
mxfp4_quantise_kernel(const T* __restrict__ x, uint32_t* __restrict__ packed, uint32_t* __restrict__ scales, int rows, int k, int terms, uint32_t pieces) {
    pdl_wait();
    pdl_trigger();
    const uint32_t chunks = (k + 255) / 256, lane = threadIdx.x & 31, at = blockIdx.x * (MXQ_THREADS / 32) + (threadIdx.x >> 5);
    if (at >= pieces) return;
    const uint32_t row = at / chunks, chunk = at % chunks;
    const bool is_in = chunk * 256 + lane * 8 < k;      // (k is a multiple of 32: a block's lanes are all in or all out)
    Eight<T> in;
    if (is_in) in.load(x + (size_t)row * k + chunk * 256 + lane * 8);
    const uint32_t term_words = (uint32_t)((rows + 127) / 128) * chunks * 256;
    uint32_t* sp = scales + ((size_t)(row / 128) * (2 * chunks) + 2 * chunk + (lane >> 4)) * 128 + (row & 31) * 4 + (row >> 5 & 3);
    uint32_t* pp = packed + ((size_t)row * k + chunk * 256 + lane * 8) / 8;
    auto scale_of = [&](uint32_t top) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int byte = scale_byte(top);
        uint32_t word = is_in ? (uint32_t)byte << (8 * (lane >> 2 & 3)) : 0u;
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if ((lane & 15) == 0) *sp = word;
        return byte;
    };
    float y[8];
    const int byte = scale_of(is_in ? in.top() : 0u);
    const float down = power_of_two(127 - byte);       // (255, NaN: the numbers behind it do not count)
    in.times(down, y);
    uint32_t held = to_e2m1x8(y);
    if (is_in) *pp = held;
    if (terms > 1) {
        float rest[8], q[8];
        in.times(1.f, rest);
        int last = byte;
        for (int t = 1; t < terms; ++t) {
            from_e2m1x8(held, q);
            const float up = power_of_two(last - 127);
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                rest[i] = last == 255 || !is_in ? 0.f : rest[i] - q[i] * up;
                top = max(top, __float_as_uint(rest[i]) & 0x7fffffffu);
            }
            sp += term_words, pp += (size_t)rows * k / 8;
            last = scale_of(top);
            const float less = power_of_two(127 - last);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = rest[i] * less;
            held = to_e2m1x8(y);
            if (is_in) *pp = held;
        }
    }
}

// The same for many rows, bound by memory as long as what a block needs besides its numbers (its scale, and where that goes) is
// done by few lanes: two are a block, sixteen numbers each, and a thread has two such halves on the way.  A row begins where the
// last one ends, so that the whole is one line of blocks.  3,584 x 18,944 and 37,888 x 3,584 from memory: float32 47 and 91 us, 6.5 and
// 6.8 TB/s; bfloat16 29 and 56, 5.9 and 6.2 (a copy 6.3 to 6.4).  With four lanes to a block, words of four scales put together by
// shuffles and four pieces to a warp bfloat16 took 44 for the first.
template <typename T>
__global__ void __launch_bounds__(MXQ_THREADS)
mxfp4_quantise_many_kernel(const T* __restrict__ x, uint32_t* __restrict__ packed, uint8_t* __restrict__ scales, int rows, int k, int terms, uint32_t halves) {
    constexpr int AT_ONCE = 2;
    pdl_wait();
    pdl_trigger();
    const uint32_t per_row = k / 32, k_tiles = 2 * ((k + 255) / 256);
    const size_t term_bytes = (size_t)((rows + 127) / 128) * k_tiles * 512, term_words = (size_t)rows * k / 8;
    Eight<T> in[AT_ONCE][2];
    uint32_t at[AT_ONCE];
    bool is_in[AT_ONCE];
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) {
        at[c] = (blockIdx.x * AT_ONCE + c) * MXQ_THREADS + threadIdx.x;
        is_in[c] = at[c] < halves;                      // (an even number: a block's two lanes are in or out together)
        if (is_in[c]) load_sixteen(x + (size_t)at[c] * 16, in[c]);
    }
#pragma unroll
    for (int c = 0; c < AT_ONCE; ++c) {
        const uint32_t block = at[c] / 2, row = block / per_row, j = block % per_row;
        uint8_t* sp = scales + (size_t)(row / 128) * k_tiles * 512 + (row & 31) * 16 + (row >> 5 & 3) * 4;
        uint32_t* pp = packed + (size_t)at[c] * 2;
        auto scale_of = [&](uint32_t top) {
            const int byte = scale_byte(max(top, __shfl_xor_sync(0xffffffffu, top, 1)));
            if (is_in[c] && (at[c] & 1) == 0) {
                sp[(j >> 2) * 512 + (j & 3)] = (uint8_t)byte;
                if (j == per_row - 1)
                    for (uint32_t i = per_row; i < 4 * k_tiles; ++i) sp[(i >> 2) * 512 + (i & 3)] = 0;
            }
            return byte;
        };
        uint32_t held[2];
        auto put = [&] {
            if (is_in[c]) *reinterpret_cast<uint2*>(pp) = make_uint2(held[0], held[1]);
        };
        int byte = scale_of(is_in[c] ? max(in[c][0].top(), in[c][1].top()) : 0u);
        float y[2][8];
        const float down = power_of_two(127 - byte);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            in[c][h].times(down, y[h]);
            held[h] = to_e2m1x8(y[h]);
        }
        put();
        if (terms > 1) {
            float rest[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h) in[c][h].times(1.f, rest[h]);
            for (int t = 1; t < terms; ++t) {
                const float up = power_of_two(byte - 127);
                uint32_t top = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float q[8];
                    from_e2m1x8(held[h], q);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        rest[h][i] = byte == 255 || !is_in[c] ? 0.f : rest[h][i] - q[i] * up;
                        top = max(top, __float_as_uint(rest[h][i]) & 0x7fffffffu);
                    }
                }
                sp += term_bytes, pp += term_words;
                byte = scale_of(top);
                const float less = power_of_two(127 - byte);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[h][i] = rest[h][i] * less;
                    held[h] = to_e2m1x8(y[h]);
                }
                put();
            }
        }
    }
}

// What add_prenorm_kernel (elementwise.cu) does, with the rows rounded to 4 bits on the way: h[t, i] += sum over parts of delta[part, t,
// i]; packed and scales hold h[t, i] * w[i] as `terms` 4-bit numbers; ss[chunk, t] = the sum of h[t, i]^2 over the chunk's MXN_CHUNK columns.
// The norm's scale per row, rsqrt(sum of ss / E + eps), commutes with the product that takes the rows, which applies it to its
// accumulators; a block's scale is made for the numbers as they are here, so nothing is lost by its coming later.  A block waits for no
// other: one round trip to L2, where the norm (a chain of a row's loads, a sum over the row, a second pass) and the rounding behind it
// were two launches.  One token of width 3,584 with four partial sums, in two terms: 4.1 us for the two, 1.8 for this; with the q/k/v
// product of 4,608 outputs behind them 8.9 and 6.2 (64 tokens: 10.3 and 9.5).
constexpr int MXN_CHUNK = 512;
constexpr int MXN_PARTS = 8;      // partial sums that a thread asks for at once
template <typename TD, typename TW>
__global__ void __launch_bounds__(MXN_CHUNK / 4)
mxfp4_add_prenorm_kernel(float* __restrict__ h, const TD* __restrict__ delta, int parts, size_t part_stride, const TW* __restrict__ w,
                         uint8_t* __restrict__ packed, uint8_t* __restrict__ scales, float* __restrict__ ss, int T, int E, int terms) {
    __shared__ float scratch[32];
    pdl_wait();
    pdl_trigger();      // (behind the wait: see mxfp4_quantise_kernel)
    const int t = blockIdx.y, lane = threadIdx.x & 31, i = blockIdx.x * MXN_CHUNK + threadIdx.x * 4;
    const bool in = i < E;                      // (E is a multiple of 32: a block's eight lanes are all in or all out)
    const size_t at = (size_t)t * E + i;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f}, d[MXN_PARTS][4];
    if (in) {
        load4(h + at, x);
        load4(w + i, y);
#pragma unroll
        for (int p = 0; p < MXN_PARTS; ++p)
            if (p < parts) load4(delta + p * part_stride + at, d[p]);
#pragma unroll
        for (int p = 0; p < MXN_PARTS; ++p)
            if (p < parts) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] += d[p][j];
            }
        for (int p = MXN_PARTS; p < parts; ++p) {
            float e[4];
            load4(delta + p * part_stride + at, e);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] += e[j];
        }
        if (parts > 0) store4(h + at, x);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] *= x[j];
    }
    const int k_tiles = 2 * ((E + 255) / 256), k_tile = i / 128;        // (a warp's columns are one tile's)
    uint8_t* sp = scales + ((size_t)(t / 128) * k_tiles + k_tile) * 512 + (t & 31) * 16 + (t >> 5 & 3) * 4;
    const size_t term_bytes = (size_t)((T + 127) / 128) * k_tiles * 512;
    for (int term = 0; term < terms; ++term) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < 8; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int byte = scale_byte(top);
        uint32_t word = in ? (uint32_t)byte << (8 * (lane >> 3)) : 0u;
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        word |= __shfl_xor_sync(0xffffffffu, word, 16);
        if (lane == 0 && k_tile < k_tiles) *reinterpret_cast<uint32_t*>(sp + term * term_bytes) = word;
        const float down = power_of_two(127 - byte), up = power_of_two(byte - 127);
        const float z[8] = {y[0] * down, y[1] * down, y[2] * down, y[3] * down, 0.f, 0.f, 0.f, 0.f};
        const uint32_t code = to_e2m1x8(z);
        if (in) *reinterpret_cast<uint16_t*>(packed + ((size_t)term * T + t) * (E / 2) + i / 2) = (uint16_t)code;
        float q[8];
        from_e2m1x8(code, q);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = byte == 255 ? 0.f : y[j] - q[j] * up;
    }
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) sq += x[j] * x[j];
    const float total = block_sum(sq, scratch);
    if (threadIdx.x == 0) ss[(size_t)blockIdx.x * T + t] = total;
}

// The numbers that packed and scales stand for: a thread takes sixteen.  Grid (terms * rows, columns).
template <typename T>
__global__ void __launch_bounds__(MXQ_THREADS)
mxfp4_values_kernel(const uint32_t* __restrict__ packed, const uint8_t* __restrict__ scales, T* __restrict__ out, int rows, int k) {
    pdl_enter(TR_MXFP4_VALUES);
    const uint32_t line = blockIdx.x, col = (blockIdx.y * blockDim.x + threadIdx.x) * 16, row = line % rows, t = line / rows, j = col / 32;
    if (col >= k) return;
    const size_t row_tiles = (rows + 127) / 128, k_tiles = 2 * ((k + 255) / 256);
    const uint2 code = *reinterpret_cast<const uint2*>(packed + ((size_t)line * k + col) / 8);
    const int byte = scales[(((size_t)t * row_tiles + row / 128) * k_tiles + j / 4) * 512 + (row % 32) * 16 + (row / 32 % 4) * 4 + j % 4];
    const float unit = byte == 255 ? __uint_as_float(0x7fc00000u) : power_of_two(byte - 127);
    float v[2][8];
    from_e2m1x8(code.x, v[0]);
    from_e2m1x8(code.y, v[1]);
    T* to = out + (size_t)line * k + col;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[h][i] *= unit;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(v[h][2 * i], v[h][2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&two);
            }
            reinterpret_cast<uint4*>(to)[h] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(to)[i] = make_float4(v[i >> 1][4 * (i & 1)], v[i >> 1][4 * (i & 1) + 1], v[i >> 1][4 * (i & 1) + 2], v[i >> 1][4 * (i & 1) + 3]);
    }
}

// ------------------------------------------------------------------------------------------------ products
// out[t][n] = sum over terms of x_term[t] . w[n].  The weights are the M side of the instruction, 128 rows of W to a tile, the
// tokens its N side (TN of them): a warp reading the accumulators then holds 32 neighbouring outputs of one token, and stores
// them as they lie, for few tokens and for many.  The tensor cores take both operands as they are stored, 64 numbers of k and
// two scales of each row to an instruction, and add up in float32; nothing is widened on the way.
//   warp 0      copies the tile of W and its scales of every step of k (256 numbers, 128 bytes of every row) into a ring of stages;
//   warp 1      brings the scales into tensor memory (every stage has columns of its own) and issues four products a term;
//   warps 2-5   the outputs: an item's accumulators into registers, then, while the next item's fill, to memory;
//   the last    copies the tiles of tokens, of all terms at once, and their scales.
// A copy costs the thread that asks for it some 150 cycles whatever its size: with one thread for all and a copy for every term a
// step of eight tokens in two terms took 1,026 cycles, and the weights came at 4.1 TB/s.
// (256 tokens, in the pairs' kernel: eight warps of outputs, half of the tokens each; stored as they were read, they kept the next
// item's products waiting 4,400 cycles of 12,200)
constexpr int mx_output_warps(int tn) { return tn > 128 ? 8 : 4; }
constexpr int mx_threads(int tn) { return 96 + 32 * mx_output_warps(tn); }
constexpr int MX_BM = 128;              // rows of W to a tile
constexpr int MX_STEP = 256;            // numbers of k to a stage
constexpr int MX_W_BYTES = MX_BM * 128;
constexpr int MX_SMEM = 220 * 1024;
constexpr int MX_MOST_STAGES = 8;

// Instruction descriptor: A and B e2m1 (type 1), scales e8m0 (bit 23), M 128; which two bytes of a word of scales are meant
// (0 or 2) stands in bits 4-5 for B and 29-30 for A.
__host__ __device__ constexpr uint32_t mx_idesc(int n, int part) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | (1u << 27) | ((uint32_t)part << 4) | ((uint32_t)part << 29);
}

// The low word of a descriptor (start address, leading offset 1); the high words are constants: 1,024 bytes (a K-major tile with the
// 128-byte swizzle, as umma_desc) or 128 (scales, without a swizzle) between groups of eight rows.
__device__ __forceinline__ uint32_t desc_low(uint32_t smem_addr) { return ((smem_addr & 0x3FFFF) >> 4) | (1u << 16); }

__device__ __forceinline__ void umma_mxfp4(uint32_t tmem_d, uint32_t low_a, uint32_t low_b, uint32_t idesc, uint32_t scale_a,
                                           uint32_t scale_b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "r"(low_a), "r"(low_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate), "n"((1024 >> 4) | (1 << 14) | (2 << 29))
        : "memory");
}

// A tile of scales (32 rows of 16 bytes, one after the other) into four columns of tensor memory, the same for all four
// quarters of its lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t tmem, uint32_t low) {
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}"
                 ::"r"(tmem), "r"(low), "n"((128 >> 4) | (1 << 14)) : "memory");
}

// A whole warp's wait: one look, which mostly is enough, then the bounded wait; the same answer for all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// splits: parts of k, written as they are, [splits][T][N].
struct MxShape {
    int T, N, splits;
    int k_steps, w_tiles, t_tiles;
    // what becomes of the sums: MX_STORE; MX_ADD, onto float32 that is there; MX_GATED, rows of W are gate and up of an output in
    // turn, out [T][N / 2] = gated_activation(gate, up, alpha, limit, shift)
    int mode;
    float alpha, limit, shift;
    // (up to 64 tokens) sums of squares [chunks][T] of the rows that mxfp4_add_prenorm_kernel wrote, or null: the sums of token t are
    // multiplied by rsqrt(sum over chunks of ss / width + eps) before all else
    const float* ss;
    int chunks, width;
    float eps;
    int w_ready;      // (few rows' kernel) W was complete before the predecessor, which rounds rows, passed its own wait
};
constexpr int MX_STORE = 0, MX_ADD = 1, MX_GATED = 2;

// An item: a tile of W, a tile of tokens and a part of k.  Items stand in this order: parts, tiles of tokens, tiles of W.
struct MxItem {
    int item, k, k1, t_tile, w_tile, split;
    __device__ __forceinline__ void at(int i, const MxShape& s, int per) {
        item = i;
        split = i % s.splits;
        const int tiles = i / s.splits;
        t_tile = tiles % s.t_tiles, w_tile = tiles / s.t_tiles;
        k = split * per, k1 = min(s.k_steps, k + per);
    }
};

template <int TN, int TERMS>
struct MxTile {
    static constexpr int X_BYTES = TN * 128;
    static constexpr int X_SCALE_TILES = (TN + 127) / 128;               // of 128 tokens
    static constexpr int X_SCALE_BYTES = X_SCALE_TILES * 1024;
    static constexpr int X_SCALE_COLS = X_SCALE_TILES * 8;
    static constexpr int SUMS = 2;                                       // accumulators in tensor memory
    // a stage: W, its scales, the tokens of every term, their scales
    static constexpr int STAGE = MX_W_BYTES + 1024 + TERMS * (X_BYTES + X_SCALE_BYTES);
    static constexpr int SCALE_COLS = 8 + TERMS * X_SCALE_COLS;
    static constexpr int FIT = (MX_SMEM - 2048) / STAGE, COLS = (512 - SUMS * TN) / SCALE_COLS;
    static constexpr int STAGES = FIT < COLS ? (FIT < MX_MOST_STAGES ? FIT : MX_MOST_STAGES) : (COLS < MX_MOST_STAGES ? COLS : MX_MOST_STAGES);
    static_assert(STAGES >= 2, "a ring of one stage");
};

// A warp's 32 outputs of COLS tokens out of tensor memory, and to where they belong: lane i holds output `col` of each token.
template <int COLS>
__device__ __forceinline__ void read_sums(uint32_t tmem, uint32_t (&v)[COLS]) {
    if constexpr (COLS < 32) {
        tmem_ld16(tmem, v);
    } else {
#pragma unroll
        for (int c = 0; c < COLS; c += 32) tmem_ld32(tmem + c, reinterpret_cast<uint32_t (&)[32]>(v[c]));
    }
}
// gated_activation (common.cuh) by the special-function unit's exponential and reciprocal (2^-22 off, which a float32 output shows and a
// bfloat16 one does not): the accurate forms, of 60 instructions, took as long as the products of a step.  Cuts and the rectifier hand NaN
// on (a block of a number that is not finite is NaN, and what is made of it must be).
__device__ __forceinline__ float min_or_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float gated_quick(float g, float u, float neg_alpha_log2, float limit, float shift) {
    if (limit > 0.f) {
        g = min_or_nan(g, limit);
        u = min_or_nan(max_or_nan(u, -limit), limit);
    }
    if (neg_alpha_log2 > 0.f) return max_or_nan(g, 0.f) * (u + shift);
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * neg_alpha_log2));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return g * r * (u + shift);
}

template <int COLS, typename TO>
__device__ __forceinline__ void store_sums(TO* out, int col, int token, const MxShape& s, const uint32_t (&v)[COLS]) {
    const int left = s.T - token;
    if (s.mode == MX_GATED) {
        // gate and up of an output are neighbouring lanes: of two tokens, the even lane finishes the first and the odd one the second
        const bool odd = col & 1;
        TO* to = out + (size_t)(token + (odd ? 1 : 0)) * (s.N / 2) + col / 2;
        const float neg_alpha_log2 = -1.4426950408889634f * s.alpha;
#pragma unroll
        for (int c = 0; c < COLS; c += 2, to += s.N) {
            const float a = __uint_as_float(v[c]), b = __uint_as_float(v[c + 1]), other = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
            if (col < s.N && c + (odd ? 1 : 0) < left) *to = from_float<TO>(gated_quick(odd ? other : a, odd ? b : other, neg_alpha_log2, s.limit, s.shift));
        }
        return;
    }
    if (col >= s.N) return;
    if constexpr (sizeof(TO) == 4) {
        if (s.mode == MX_ADD) {
            // (an addition in L2, which nothing waits for; every number gets one)
            float* to = (float*)out + (size_t)token * s.N + col;
#pragma unroll
            for (int c = 0; c < COLS; ++c, to += s.N)
                if (c < left) asm volatile("red.global.add.f32 [%0], %1;" ::"l"(to), "f"(__uint_as_float(v[c])) : "memory");
            return;
        }
    }
    TO* to = out + (size_t)token * s.N + col;
    if (left >= COLS) {
#pragma unroll
        for (int c = 0; c < COLS; ++c, to += s.N) *to = from_float<TO>(__uint_as_float(v[c]));
        return;
    }
    // (eight tokens at a time without a branch for every one: with one, 256 tokens took 18,900 cycles, twice the products' time)
#pragma unroll
    for (int c = 0; c < COLS; c += 8) {
        if (c + 8 <= left) {
#pragma unroll
            for (int i = 0; i < 8; ++i, to += s.N) *to = from_float<TO>(__uint_as_float(v[c + i]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i, to += s.N)
                if (c + i < left) *to = from_float<TO>(__uint_as_float(v[c + i]));
        }
    }
}

// What the issuing warp does for a step besides its products is what the products wait for: with remainders by a number of stages
// known at run time, 64-bit descriptors and waits that always vote it took 850 cycles a step, whatever the products; unrolled over
// the stages 800 (the code no longer fits the nearest instruction cache); so, with the terms alone unrolled, it takes 423
// cycles for few tokens in one term and 596 in two.
template <int TN, int TERMS, typename TO>
__global__ void __launch_bounds__(mx_threads(TN), 1)
mxfp4_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_w,
                  const uint8_t* __restrict__ w_scales, TO* __restrict__ out, const MxShape s, int* __restrict__ status) {
    using Tile = MxTile<TN, TERMS>;
    constexpr int SUMS = Tile::SUMS, STAGE = Tile::STAGE, STAGES = Tile::STAGES;
    constexpr int OUT_WARPS = mx_output_warps(TN), X_WARP = 2 + OUT_WARPS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + STAGES * STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* done = empty + STAGES;                // [SUMS]: an item's accumulators are complete
    uint64_t* taken = done + SUMS;                  // [SUMS]: and have been read
    uint32_t* tmem_slot = (uint32_t*)(taken + SUMS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    float* row_scale = (float*)(tmem_slot + 2);     // [TN]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 2);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < SUMS; ++i) {
            mbar_init(&done[i], 1);
            mbar_init(&taken[i], OUT_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    const int items = s.w_tiles * s.t_tiles * s.splits;
    const int per = (s.k_steps + s.splits - 1) / s.splits;
    MxItem it;
    it.at(blockIdx.x, s, per);

    if (warp == 0 || warp == X_WARP) {
        // ---------------------------------------------------- copies
        // (w_ready: only the tokens wait.  A kernel that rounds rows lets this one start behind its own wait, so that weights written
        // ahead of it are there; rounding may be rounding of these very weights where no rounding of tokens stands in between)
        if (warp == X_WARP || !s.w_ready) pdl_wait();
        uint32_t st = 0, parity = 1;
        while (it.item < items) {
            if (!warp_wait(&empty[st], parity, abort_flag)) break;        // (a fresh barrier's phase ahead of its first counts as over)
            if (elect_one()) {
                uint8_t* to = smem + st * STAGE;
                if (warp == 0) {
                    mbar_expect_tx(&full[st], MX_W_BYTES + 1024);
                    tma_load_2d(to, &map_w, it.k * 128, it.w_tile * MX_BM, &full[st]);
                    bulk_load(to + MX_W_BYTES, w_scales + ((size_t)it.w_tile * s.k_steps + it.k) * 1024, 1024, &full[st]);
                } else {
                    mbar_expect_tx(&full[st], STAGE - MX_W_BYTES - 1024);
                    tma_load_3d(to + MX_W_BYTES + 1024, &map_x, it.k * 128, it.t_tile * TN, 0, &full[st]);
                    tma_load_3d(to + MX_W_BYTES + 1024 + TERMS * Tile::X_BYTES, &map_xs, it.k * 256, it.t_tile * Tile::X_SCALE_TILES, 0, &full[st]);
                }
            }
            __syncwarp();
            if (++st == STAGES) st = 0, parity ^= 1;
            if (++it.k == it.k1) it.at(it.item + gridDim.x, s, per);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------- products
        uint32_t st = 0, parity = 0, sums = 0, sums_parity = 1;
        bool ok = true;
        const uint32_t low = desc_low(smem_u32(smem));
        while (ok && it.item < items) {
            if (!(ok = warp_wait(&taken[sums], sums_parity, abort_flag))) break;
            const uint32_t d = tmem + sums * TN;
            uint32_t accumulate = 0;
            for (; it.k < it.k1; ++it.k) {
                if (!(ok = warp_wait(&full[st], parity, abort_flag))) break;
                tc_fence_after();
                const uint32_t w_at = low + st * (STAGE >> 4), sw = tmem + SUMS * TN + st * Tile::SCALE_COLS;
                if (elect_one()) {
                    scales_to_tmem(sw, w_at + (MX_W_BYTES >> 4));
                    scales_to_tmem(sw + 4, w_at + ((MX_W_BYTES + 512) >> 4));
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t x_at = w_at + ((MX_W_BYTES + 1024 + t * Tile::X_BYTES) >> 4), sx = sw + 8 + t * Tile::X_SCALE_COLS;
                        const uint32_t xs_at = w_at + ((MX_W_BYTES + 1024 + TERMS * Tile::X_BYTES + t * Tile::X_SCALE_BYTES) >> 4);
#pragma unroll
                        for (int r = 0; r < Tile::X_SCALE_TILES; ++r)
#pragma unroll
                            for (int a = 0; a < 2; ++a)      // (an instruction's scales of 256 tokens stand side by side)
                                scales_to_tmem(sx + a * 4 * Tile::X_SCALE_TILES + r * 4, xs_at + r * 64 + a * 32);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma_mxfp4(d, w_at + 2 * kk, x_at + 2 * kk, mx_idesc(TN, 2 * (kk & 1)), sw + 4 * (kk >> 1),
                                       sx + 4 * Tile::X_SCALE_TILES * (kk >> 1), t > 0 || kk > 0 ? 1u : accumulate);
                    }
                    umma_commit(&empty[st]);
                }
                __syncwarp();
                accumulate = 1;
                if (++st == STAGES) st = 0, parity ^= 1;
            }
            if (!ok) break;
            if (elect_one()) umma_commit(&done[sums]);
            __syncwarp();
            if (++sums == SUMS) sums = 0, sums_parity ^= 1;
            it.at(it.item + gridDim.x, s, per);
        }
    } else {
        // ---------------------------------------------------- outputs
        const int quarter = warp & 3;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        bool ok = true;
        if (s.ss) {      // (one tile of tokens)
            pdl_wait();
            const int t = threadIdx.x - 64;
            if (t < TN) {
                float total = 0.f;
                for (int c0 = 0; c0 < s.chunks; c0 += 8) {
                    float part[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) part[i] = c0 + i < s.chunks && t < s.T ? s.ss[(size_t)(c0 + i) * s.T + t] : 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) total += part[i];
                }
                row_scale[t] = rsqrtf(total / (float)s.width + s.eps);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(OUT_WARPS * 32) : "memory");
        }
        for (int turn = 0; it.item < items; ++turn, it.at(it.item + gridDim.x, s, per)) {
            ok = warp_wait(&done[turn % SUMS], (turn / SUMS) & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            constexpr int COLS = TN / (OUT_WARPS / 4);
            const int first = (warp - 2) / 4 * COLS;
            uint32_t v[COLS];
            read_sums<COLS>(tmem + (turn % SUMS) * TN + lane_addr + first, v);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&taken[turn % SUMS]);
            if (s.ss) {
#pragma unroll
                for (int c = 0; c < COLS; ++c) v[c] = __float_as_uint(__uint_as_float(v[c]) * row_scale[first + c]);
            }
            store_sums<COLS>(out + (size_t)it.split * s.T * s.N, it.w_tile * MX_BM + quarter * 32 + lane, it.t_tile * TN + first, s, v);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 32; ++i) __nanosleep(2000);     // copies on their way may still land
        if (threadIdx.x == 0 && status) atomicExch(status, 10);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// The sums of a product's parts [n_parts][n], in their order, and what MxShape's mode makes of them: two outputs (or the gate and the up
// of one) to a thread.  The parts stay in L2.  As its blocks' last deed the product's kernel did this in 10 us and more for 128 tokens
// of a tile: a fence, a count and a chain of loads by the few warps of the last block, in code that runs once and comes from memory.
template <typename TO>
__global__ void __launch_bounds__(256)
mxfp4_join_kernel(const float* __restrict__ parts, TO* __restrict__ out, size_t n, int n_parts, int mode, float alpha, float limit, float shift) {
    pdl_enter(TR_MXFP4_JOIN);
    const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 2;
    if (at >= n) return;
    const bool both = at + 1 < n;
    float a = 0.f, b = 0.f;
    for (int p = 0; p < n_parts; p += 8) {
        float x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (p + i < n_parts) {
                const float* from = parts + (p + i) * n + at;       // (n may be odd: no pairs)
                x[i] = from[0];
                y[i] = both ? from[1] : 0.f;
            }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (p + i < n_parts) a += x[i], b += y[i];
    }
    if (mode == MX_GATED) {      // (N is even)
        out[at / 2] = from_float<TO>(gated_quick(a, b, -1.4426950408889634f * alpha, limit, shift));
        return;
    }
    if constexpr (sizeof(TO) == 4) {
        if (mode == MX_ADD) {
            a += out[at];
            if (both) b += out[at + 1];
        }
    }
    out[at] = from_float<TO>(a);
    if (both) out[at + 1] = from_float<TO>(b);
}

// ------------------------------------------------------------------------------------------------ products of many rows
// Two SMs share a tile of 256 rows of W and TN tokens (cta_group::2): each holds 128 of the rows of W and half of the tokens, and its
// accumulators are its own rows' for all of the tokens.  An SM then fetches, for TN = 256 and one term, 35 KB a step where a tile of
// its own of 128 x 256 takes 52: at 128 cycles a product the SMs together would ask L2 for 15 KB a cycle, of which it gives some
// 8.  The scales of the tokens are wanted whole on both sides.
//   warp 0      of each side copies W's rows and their scales, the last warp the tokens and their scales;
//   warp 1      of the first side issues copies of scales and products for both; that of the second says there when its stage is full;
//   the others  store their side's rows.
// A stage, and the accumulators, are free when both sides have said so.
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives on the barrier at the same place in the cluster's first block.  What it says is that copies have landed or tensor memory was
// read, not that this thread's own writes to memory are there: a release to the whole cluster waits for those, and took 1,800 cycles.
__device__ __forceinline__ void arrive_at_first(uint64_t* bar) {
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, 0;\n\tmbarrier.arrive.shared::cluster.b64 _, [r];\n\t}"
                 ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pair_commit(uint64_t* bar) {        // arrives on both sides
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void pair_umma_mxfp4(uint32_t tmem_d, uint32_t low_a, uint32_t low_b, uint32_t idesc, uint32_t scale_a,
                                                uint32_t scale_b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a, b, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "r"(low_a), "r"(low_b), "r"(idesc), "r"(scale_a), "r"(scale_b), "r"(accumulate), "n"((1024 >> 4) | (1 << 14) | (2 << 29))
        : "memory");
}
__device__ __forceinline__ void pair_scales_to_tmem(uint32_t tmem, uint32_t low) {
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}"
                 ::"r"(tmem), "r"(low), "n"((128 >> 4) | (1 << 14)) : "memory");
}
__host__ __device__ constexpr uint32_t mx_pair_idesc(int n, int part) { return (mx_idesc(n, part) & ~(1u << 27)) | (1u << 28); }      // M 256

template <int TN, int TERMS>
struct MxPairTile {
    static constexpr int X_BYTES = TN / 2 * 128;
    static constexpr int X_SCALE_TILES = TN / 128, X_SCALE_BYTES = X_SCALE_TILES * 1024, X_SCALE_COLS = X_SCALE_TILES * 8;
    static constexpr int SUMS = TN <= 128 ? 2 : 1;
    static constexpr int STAGE = MX_W_BYTES + 1024 + TERMS * (X_BYTES + X_SCALE_BYTES);
    static constexpr int SCALE_COLS = 8 + TERMS * X_SCALE_COLS;
    static constexpr int FIT = (MX_SMEM - 2048) / STAGE, COLS = (512 - SUMS * TN) / SCALE_COLS;
    static constexpr int STAGES = FIT < COLS ? (FIT < MX_MOST_STAGES ? FIT : MX_MOST_STAGES) : (COLS < MX_MOST_STAGES ? COLS : MX_MOST_STAGES);
    static_assert(STAGES >= 2, "a ring of one stage");
};

template <int TN, int TERMS, typename TO>
__global__ void __launch_bounds__(mx_threads(TN), 1)
mxfp4_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_xs, const __grid_constant__ CUtensorMap map_w,
                  const uint8_t* __restrict__ w_scales, TO* __restrict__ out, const MxShape s, int* __restrict__ status) {
    using Tile = MxPairTile<TN, TERMS>;
    constexpr int SUMS = Tile::SUMS, STAGE = Tile::STAGE, STAGES = Tile::STAGES;
    constexpr int OUT_WARPS = mx_output_warps(TN), X_WARP = 2 + OUT_WARPS;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* full = (uint64_t*)(smem + STAGES * STAGE);
    uint64_t* empty = full + STAGES;
    uint64_t* done = empty + STAGES;
    uint64_t* taken = done + SUMS;
    uint32_t* tmem_slot = (uint32_t*)(taken + SUMS);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t side = cluster_rank();
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], side == 0 ? 3 : 2);      // the two copying warps; on the first side, the second side's word too
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < SUMS; ++i) {
            mbar_init(&done[i], 1);
            mbar_init(&taken[i], 2 * OUT_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    const int items = s.w_tiles * s.t_tiles * s.splits, pairs = gridDim.x / 2;      // (w_tiles: of 256 rows here)
    const int per = (s.k_steps + s.splits - 1) / s.splits;
    MxItem it;
    it.at(blockIdx.x / 2, s, per);

    if (warp == 0 || warp == X_WARP) {
        // ---------------------------------------------------- copies
        if (warp == X_WARP) pdl_wait();
        uint32_t st = 0, parity = 1;
        // (a last tile of W may have one half only: the other's rows come as zeros, and its scales are any tile's)
        const int last_tile = (s.N + MX_BM - 1) / MX_BM - 1;
        while (it.item < items) {
            if (!warp_wait(&empty[st], parity, abort_flag)) break;
            if (elect_one()) {
                uint8_t* to = smem + st * STAGE;
                if (warp == 0) {
                    const int w_tile = 2 * it.w_tile + side;
                    mbar_expect_tx(&full[st], MX_W_BYTES + 1024);
                    tma_load_2d(to, &map_w, it.k * 128, w_tile * MX_BM, &full[st]);
                    bulk_load(to + MX_W_BYTES, w_scales + ((size_t)min(w_tile, last_tile) * s.k_steps + it.k) * 1024, 1024, &full[st]);
                } else {
                    mbar_expect_tx(&full[st], STAGE - MX_W_BYTES - 1024);
                    tma_load_3d(to + MX_W_BYTES + 1024, &map_x, it.k * 128, it.t_tile * TN + side * (TN / 2), 0, &full[st]);
                    tma_load_3d(to + MX_W_BYTES + 1024 + TERMS * Tile::X_BYTES, &map_xs, it.k * 256, it.t_tile * Tile::X_SCALE_TILES, 0, &full[st]);
                }
            }
            __syncwarp();
            if (++st == STAGES) st = 0, parity ^= 1;
            if (++it.k == it.k1) it.at(it.item + pairs, s, per);
        }
    } else if (warp == 1 && side == 1) {
        // ---------------------------------------------------- the second side's word that a stage is full
        uint32_t st = 0, parity = 0;
        while (it.item < items) {
            if (!warp_wait(&full[st], parity, abort_flag)) break;
            if (elect_one()) arrive_at_first(&full[st]);
            __syncwarp();
            if (++st == STAGES) st = 0, parity ^= 1;
            if (++it.k == it.k1) it.at(it.item + pairs, s, per);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------- products
        uint32_t st = 0, parity = 0, sums = 0, sums_parity = 1;
        bool ok = true;
        const uint32_t low = desc_low(smem_u32(smem));
        while (ok && it.item < items) {
            if (!(ok = warp_wait(&taken[sums], sums_parity, abort_flag))) break;
            tc_fence_after();
            const uint32_t d = tmem + sums * TN;
            uint32_t accumulate = 0;
            for (; it.k < it.k1; ++it.k) {
                if (!(ok = warp_wait(&full[st], parity, abort_flag))) break;
                tc_fence_after();
                const uint32_t w_at = low + st * (STAGE >> 4), sw = tmem + SUMS * TN + st * Tile::SCALE_COLS;
                if (elect_one()) {
                    pair_scales_to_tmem(sw, w_at + (MX_W_BYTES >> 4));
                    pair_scales_to_tmem(sw + 4, w_at + ((MX_W_BYTES + 512) >> 4));
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) {
                        const uint32_t x_at = w_at + ((MX_W_BYTES + 1024 + t * Tile::X_BYTES) >> 4), sx = sw + 8 + t * Tile::X_SCALE_COLS;
                        const uint32_t xs_at = w_at + ((MX_W_BYTES + 1024 + TERMS * Tile::X_BYTES + t * Tile::X_SCALE_BYTES) >> 4);
#pragma unroll
                        for (int r = 0; r < Tile::X_SCALE_TILES; ++r)
#pragma unroll
                            for (int a = 0; a < 2; ++a)
                                pair_scales_to_tmem(sx + a * 4 * Tile::X_SCALE_TILES + r * 4, xs_at + r * 64 + a * 32);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            pair_umma_mxfp4(d, w_at + 2 * kk, x_at + 2 * kk, mx_pair_idesc(TN, 2 * (kk & 1)), sw + 4 * (kk >> 1),
                                            sx + 4 * Tile::X_SCALE_TILES * (kk >> 1), t > 0 || kk > 0 ? 1u : accumulate);
                    }
                    pair_commit(&empty[st]);
                }
                __syncwarp();
                accumulate = 1;
                if (++st == STAGES) st = 0, parity ^= 1;
            }
            if (!ok) break;
            if (elect_one()) pair_commit(&done[sums]);
            __syncwarp();
            if (++sums == SUMS) sums = 0, sums_parity ^= 1;
            it.at(it.item + pairs, s, per);
        }
    } else {
        // ---------------------------------------------------- outputs
        const int quarter = warp & 3;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        for (int turn = 0; it.item < items; ++turn, it.at(it.item + pairs, s, per)) {
            if (!warp_wait(&done[turn % SUMS], (turn / SUMS) & 1, abort_flag)) break;
            tc_fence_after();
            constexpr int COLS = TN / (OUT_WARPS / 4);
            const int first = (warp - 2) / 4 * COLS;
            uint32_t v[COLS];
            read_sums<COLS>(tmem + (turn % SUMS) * TN + lane_addr + first, v);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at_first(&taken[turn % SUMS]);
            store_sums<COLS>(out + (size_t)it.split * s.T * s.N, (2 * it.w_tile + side) * MX_BM + quarter * 32 + lane, it.t_tile * TN + first, s, v);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 32; ++i) __nanosleep(2000);     // copies on their way may still land
        if (threadIdx.x == 0 && status) atomicExch(status, 10);
    }
    cluster_sync();         // (neither side's memory goes while the other may still reach it)
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Rows of `cols` elements (bytes, or words of 32 bits) in planes: boxes of box_cols x box_rows x box_planes, with the 128-byte
// swizzle or as they lie; what lies outside comes as zeros.
static int plane_map(CUtensorMap* map, CUtensorMapDataType type, int size, const void* base, long long cols, long long rows, long long planes, int box_cols,
                     int box_rows, int box_planes, bool swizzle) {
    EncodeTiled enc = encode_tiled();
    if (!enc) return AIR_ERR_BAD_ARGUMENT;
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)(cols * size), (cuuint64_t)(cols * rows * size)};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, (cuuint32_t)box_planes};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r = enc(map, type, box_planes ? 3 : 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : 200000 + (int)r;
}

struct MxCall {
    const void *packed, *scales, *w;
    const uint8_t* w_scales;
    void* out;
    int T, N, K, splits;
    int sms;
    int* status;
    cudaStream_t stream;
    int mode;
    float alpha, limit, shift;
    const float* ss;
    int chunks;
    float eps;
    int w_ready;
};

// pair: 0, a block for itself; 1, two share a tile (cluster of two).
template <typename Tile, int TN, int TERMS, typename TO, typename Kernel>
static int launch_mxfp4(Kernel kernel, int pair, int x_rows, const MxCall& c) {
    const int rows = MX_BM << pair, units = c.sms >> pair;
    const MxShape s{c.T, c.N, c.splits, (c.K + MX_STEP - 1) / MX_STEP, (c.N + rows - 1) / rows, (c.T + TN - 1) / TN,
                    c.mode, c.alpha, c.limit, c.shift, c.ss, c.chunks, c.K, c.eps, c.w_ready};
    // (a part without a step of k would leave its sums unwritten)
    const int per = (s.k_steps + c.splits - 1) / c.splits;
    const long long items = (long long)s.w_tiles * s.t_tiles * c.splits;
    if ((c.splits - 1) * per >= s.k_steps || items > 0x3fffffffll || units < 1) return AIR_ERR_BAD_ARGUMENT;
    CUtensorMap mx, mxs, mw;
    int rc = plane_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.packed, c.K / 2, c.T, TERMS, 128, x_rows, TERMS, true);
    if (!rc)
        rc = plane_map(&mxs, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, c.scales, (long long)s.k_steps * 256, (c.T + 127) / 128, TERMS, 256, Tile::X_SCALE_TILES,
                       TERMS, false);
    if (!rc) rc = plane_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, c.w, c.K / 2, c.N, 1, 128, MX_BM, 0, true);
    if (rc) return rc;
    const size_t smem = 1024 + (size_t)Tile::STAGES * Tile::STAGE + 512;      // (barriers, and 64 tokens' scales)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((int)(items < units ? items : units) << pair);
    cfg.blockDim = dim3(mx_threads(TN));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = pdl_enabled() ? attr : attr + 1;
    cfg.numAttrs = (pdl_enabled() ? 1 : 0) + pair;
    return launch_counted(cfg, kernel, mx, mxs, mw, c.w_scales, (TO*)c.out, s, c.status);
}
template <int TN, int TERMS, typename TO>
static int launch_mxfp4_alone(const MxCall& c) {
    return launch_mxfp4<MxTile<TN, TERMS>, TN, TERMS, TO>(mxfp4_gemm_kernel<TN, TERMS, TO>, 0, TN, c);
}
template <int TN, int TERMS, typename TO>
static int launch_mxfp4_pair(const MxCall& c) {
    return launch_mxfp4<MxPairTile<TN, TERMS>, TN, TERMS, TO>(mxfp4_pair_kernel<TN, TERMS, TO>, 1, TN / 2, c);
}

// Which kernel takes a product, and in how many parts it cuts k where its sums are to be joined: the least of rounds of items over
// the SMs (or pairs of them), times an item's steps, times what a step takes, and for parts the launch that joins them and their way to
// L2 and back.  Where all SMs are busy a step of 128 tokens takes 0.28, 0.40 and 0.56 us with one, two and three terms, of 256 0.46, 0.77
// and 1.14 (a fifth of the pairs alone: half of that, since L2 gives them more), of up to 64 0.22, 0.31 and 0.42, which is issuing.
// Measured, us, tiles of 128 and of 256 tokens: 2,048 x 37,888 x 3,584 125 / 104, two terms 179 / 173, three 252 / 256; 2,048 x 5,120 x
// 13,824 80 / 73, 120 / 134, 177 / 198.  One part and several: 128 x 640 x 2,048 6.6 / 7.0 (8), 128 x 4,608 x 3,584 8.0 / 9.5 (4), 256 x
// 5,120 x 13,824 18.6 / 20.4 (3), 129 of them 18.5 / 17.4; 301 x 3,584 x 18,944 in two terms 34.5 / 32.6 (3), 128 x 3,584 x 18,944 in one
// 14.9 with five.  Few rows in two terms, their rounding included, with 1, 2, 4, 5, 7 and 8 parts (- where one would have no step), what is taken
// in brackets: 1 x 4,608 x 3,584 8.0, 7.1, [6.5], 7.0, 6.7, -; 8 of them 8.2, 7.5, [6.7], 7.2, 6.8, -; 64 [9.2], 9.1, 8.4, 9.6, 9.0, -; 1 x 3,584 x
// 3,584 8.1, 7.3, 6.4, [6.4], 6.8, -; 1 x 640 x 2,048 [6.2], 6.2, 5.7, -, -, 5.2; 64 of them [6.9], 6.9, 6.5, -, -, 6.2; 1 x 3,584 x 18,944 26.4, 16.6,
// 11.2, [10.2], 12.3, 11.7; 64 of them 30.9, 20.5, 15.2, [13.8], 18.0, 17.6; 1 x 512 x 8,192 13.5, 9.6, 7.6, 7.3, 6.6, 6.5, [6.4 (16)]: within a fifth of
// the best of them.
struct MxPlan {
    int tn, pair, parts;
};
static MxPlan mx_plan(int T, int N, int K, int terms, int sms) {
    constexpr double STEP[3][3] = {{0.22, 0.31, 0.42}, {0.28, 0.40, 0.56}, {0.46, 0.77, 1.14}};
    MxPlan best{T <= 16 ? 16 : T <= 32 ? 32 : 64, T > 64, 1};
    const int w_tiles = (N + (MX_BM << best.pair) - 1) / (MX_BM << best.pair), units = sms >> best.pair, steps = (K + MX_STEP - 1) / MX_STEP;
    double least = 1e30;
    for (int tn = best.pair ? 128 : best.tn; tn <= (T > 128 ? 256 : best.pair ? 128 : best.tn); tn *= 2)
        for (int parts = 1; parts <= 16 && parts <= steps; ++parts) {
            const int per = (steps + parts - 1) / parts;
            if ((parts - 1) * per >= steps) continue;      // (a part without a step)
            const double mb = parts * 4e-6 * T * N;
            if (parts > 1 && mb > 64) break;
            const long long rounds = ((long long)w_tiles * ((T + tn - 1) / tn) * parts + units - 1) / units;
            const double busy = rounds > 1 || !best.pair ? 1.0 : (double)w_tiles * ((T + tn - 1) / tn) * parts / units;
            const double us = rounds * per * STEP[tn > 128 ? 2 : tn > 64 ? 1 : 0][terms - 1] * (0.45 + 0.55 * busy) + (parts > 1 ? 2.5 + 0.35 * mb : 0.0);
            if (us < least) least = us, best = {tn, best.pair, parts};
        }
    return best;
}

template <int TERMS, typename TO>
static int launch_mxfp4_rows(const MxPlan& p, const MxCall& c) {
    if (p.pair) return p.tn == 256 ? launch_mxfp4_pair<256, TERMS, TO>(c) : launch_mxfp4_pair<128, TERMS, TO>(c);
    return p.tn == 16 ? launch_mxfp4_alone<16, TERMS, TO>(c) : p.tn == 32 ? launch_mxfp4_alone<32, TERMS, TO>(c) : launch_mxfp4_alone<64, TERMS, TO>(c);
}

template <typename TO>
static int launch_mxfp4_terms(const MxPlan& p, int terms, const MxCall& c) {
    return terms == 1 ? launch_mxfp4_rows<1, TO>(p, c) : terms == 2 ? launch_mxfp4_rows<2, TO>(p, c) : launch_mxfp4_rows<3, TO>(p, c);
}

template <typename TO>
static int launch_join(const float* parts, TO* out, int T, int N, int n_parts, int mode, float alpha, float limit, float shift, cudaStream_t stream) {
    const long long pairs = ((long long)T * N + 1) / 2, blocks = (pairs + 255) / 256;
    if (blocks > 0x7fffffffll) return AIR_ERR_BAD_ARGUMENT;
    return launch(mxfp4_join_kernel<TO>, (int)blocks, 256, 0, stream, parts, out, (size_t)T * N, n_parts, mode, alpha, limit, shift);
}

// From how many pieces of 256 numbers on two lanes take a block.  us with four lanes and two, bfloat16, one term and two: 64 x 3,584 1.5 /
// 1.6, 1.7 / 2.3; 301 x 3,584 2.0 / 1.7, 2.5 / 2.4; 1,000 x 3,584 3.3 / 3.1, 5.4 / 5.7; 2,048 x 3,584 5.6 / 3.9, 9.9 / 7.7; 2,048 x 18,944
// 25 / 16, 48 / 32.
constexpr long long MXQ_MANY = 4096;
template <typename T>
static int launch_quantise(const void* x, void* packed, void* scales, int rows, int k, int terms, cudaStream_t stream) {
    const long long pieces = (long long)rows * ((k + 255) / 256);
    if (pieces > 0x3fffffffll) return AIR_ERR_BAD_ARGUMENT;
    const long long halves = (long long)rows * (k / 16);
    if (pieces >= MXQ_MANY && halves < 0xffff0000ll && ((uintptr_t)x & 31) == 0)
        return launch(mxfp4_quantise_many_kernel<T>, (int)((halves + 2 * MXQ_THREADS - 1) / (2 * MXQ_THREADS)), MXQ_THREADS, 0, stream, (const T*)x,
                      (uint32_t*)packed, (uint8_t*)scales, rows, k, terms, (uint32_t)halves);
    return launch(mxfp4_quantise_kernel<T>, (int)((pieces + MXQ_THREADS / 32 - 1) / (MXQ_THREADS / 32)), MXQ_THREADS, 0, stream, (const T*)x,
                  (uint32_t*)packed, (uint32_t*)scales, rows, k, terms, (uint32_t)pieces);
}

}  // namespace air

static bool mx_fits(int rows, int k, int terms) { return rows >= 0 && k >= 32 && k % 32 == 0 && terms >= 1 && terms <= 3; }

// x [rows, k] float32 or bfloat16 -> packed [terms, rows, k / 2], scales (see the head of this file).
AIR_API int air_mxfp4_quantise(const void* x, int dtype, void* packed, void* scales, int rows, int k, int terms, cudaStream_t stream) {
    if (!mx_fits(rows, k, terms) || (((uintptr_t)x | (uintptr_t)packed | (uintptr_t)scales) & 15)) return AIR_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    AIR_DISPATCH(dtype, T, { return air::launch_quantise<T>(x, packed, scales, rows, k, terms, stream); });
}

// out [terms, rows, k] float32 or bfloat16.
AIR_API int air_mxfp4_values(const void* packed, const void* scales, void* out, int dtype, int rows, int k, int terms, cudaStream_t stream) {
    if (!mx_fits(rows, k, terms) || (((uintptr_t)out | (uintptr_t)packed | (uintptr_t)scales) & 15)) return AIR_ERR_BAD_ARGUMENT;
    if (rows == 0) return 0;
    const long long lines = (long long)terms * rows;
    const int threads = k / 16 < air::MXQ_THREADS ? (k / 16 + 31) / 32 * 32 : air::MXQ_THREADS, columns = (k / 16 + threads - 1) / threads;
    if (lines > 0x7fffffffll || columns > 65535) return AIR_ERR_BAD_ARGUMENT;
    AIR_DISPATCH(dtype, T, {
        return air::launch(air::mxfp4_values_kernel<T>, dim3((int)lines, columns), threads, 0, stream, (const uint32_t*)packed,
                           (const uint8_t*)scales, (T*)out, rows, k);
    });
}

namespace air {
// What a product keeps in its working memory: the rounded tokens and their scales, and where parts of k are joined the parts.
struct MxMemory {
    size_t packed, scales, parts, bytes;      // offsets
};
static MxMemory mx_memory(int T, int N, int K, int terms, int join) {
    MxMemory m{};
    auto put = [&](size_t& at, size_t n) {
        at = m.bytes;
        m.bytes += (n + 255) / 256 * 256;
    };
    put(m.packed, (size_t)terms * T * (K / 2));
    put(m.scales, (size_t)terms * ((T + 127) / 128) * ((K + 255) / 256) * 1024);
    put(m.parts, join > 1 ? (size_t)join * T * N * sizeof(float) : 0);
    return m;
}
}  // namespace air

// Bytes of working memory for air_mxfp4_linear of these sizes, and in how many parts a product of complete sums cuts k.
AIR_API int air_mxfp4_need(int T, int N, int K, int terms, int splits, int sms, long long* need) {
    if (!mx_fits(T, K, terms) || T < 1 || N < 1 || splits < 1 || sms < 2) return AIR_ERR_BAD_ARGUMENT;
    const air::MxPlan p = air::mx_plan(T, N, K, terms, sms);
    need[0] = (long long)air::mx_memory(T, N, K, terms, splits == 1 ? p.parts : 1).bytes;
    need[1] = p.parts;
    return 0;
}

// x [T, K] float32 or bfloat16, rounded to `terms` terms; out [T, N] float32 or bfloat16 = x W^T with w [N, K / 2] and w_scales held in
// 4 bits; memory: air_mxfp4_need's bytes, on a boundary of 256, that nothing else uses until the call has run.  splits > 1 (up to 64
// rows, float32, mode 0): out [splits, T, N], sums over parts of k.  mode, alpha, limit, shift: MxShape.
AIR_API int air_mxfp4_linear(const void* x, int dtype, void* memory, const void* w, const void* w_scales, void* out, int out_dtype, int T, int N,
                             int K, int terms, int splits, int mode, float alpha, float limit, float shift, int sms, int* status,
                             cudaStream_t stream) {
    using namespace air;
    if (!mx_fits(T, K, terms) || N < 1 || splits < 1 || (splits > 1 && (out_dtype != AIR_F32 || T > 64 || mode != MX_STORE)) || sms < 2 ||
        mode < MX_STORE || mode > MX_GATED || (mode == MX_ADD && out_dtype != AIR_F32) || (mode == MX_GATED && N % 2) ||
        (((uintptr_t)x | (uintptr_t)w | (uintptr_t)w_scales) & 15) || ((uintptr_t)memory & 255))
        return AIR_ERR_BAD_ARGUMENT;
    if (T == 0) return 0;
    const MxPlan p = mx_plan(T, N, K, terms, sms);
    const int join = splits == 1 ? p.parts : 1;
    const MxMemory m = mx_memory(T, N, K, terms, join);
    uint8_t* at = (uint8_t*)memory;
    void *packed = at + m.packed, *scales = at + m.scales;
    int rc = dtype == AIR_F32 ? launch_quantise<float>(x, packed, scales, T, K, terms, stream)
             : dtype == AIR_BF16 ? launch_quantise<__nv_bfloat16>(x, packed, scales, T, K, terms, stream) : AIR_ERR_BAD_ARGUMENT;
    if (rc) return rc;
    MxCall c{packed, scales, w, (const uint8_t*)w_scales, out, T, N, K, splits, sms, status, stream, mode, alpha, limit, shift, nullptr, 0, 0.f, 1};
    if (join > 1) {
        c.out = at + m.parts, c.splits = join, c.mode = MX_STORE;
        rc = launch_mxfp4_terms<float>(p, terms, c);
        if (rc) return rc;
    }
    AIR_DISPATCH(out_dtype, TO, {
        if (join > 1)
            return launch_join<TO>((const float*)(at + m.parts), (TO*)out, T, N, join, mode, alpha, limit, shift, stream);
        return launch_mxfp4_terms<TO>(p, terms, c);
    });
}

// h [T, E] += delta ([T, E], or `parts` of them, or null); packed, scales: h * w as `terms` 4-bit numbers; ss float32 [chunks of 512
// columns][T]: the rows of an RMSNorm short of their scale (mxfp4_add_prenorm_kernel).
AIR_API int air_mxfp4_add_prenorm(float* h, const void* delta, int delta_dtype, int parts, const void* w, int w_dtype, void* packed, void* scales,
                                  float* ss, int T, int E, int terms, cudaStream_t stream) {
    using namespace air;
    auto unaligned = [](const void* p, int dtype) { return ((uintptr_t)p & (dtype == AIR_F32 ? 15 : 7)) != 0; };      // (four numbers at a time)
    if (!mx_fits(T, E, terms) || T > 65535 || parts < 0 || !h || !w || !ss || unaligned(h, AIR_F32) || unaligned(delta, delta_dtype) ||
        unaligned(w, w_dtype) || (((uintptr_t)packed | (uintptr_t)scales) & 15))
        return AIR_ERR_BAD_ARGUMENT;
    if (T == 0) return 0;
    if (!delta) parts = 0;
    const dim3 grid((E + MXN_CHUNK - 1) / MXN_CHUNK, T);
    AIR_DISPATCH(delta ? delta_dtype : AIR_F32, TD, AIR_DISPATCH(w_dtype, TW, {
        return launch(mxfp4_add_prenorm_kernel<TD, TW>, grid, MXN_CHUNK / 4, 0, stream, h, (const TD*)delta, parts, (size_t)T * E, (const TW*)w,
                      (uint8_t*)packed, (uint8_t*)scales, ss, T, E, terms);
    }));
    return 0;
}

// air_mxfp4_linear for up to 64 rows that air_mxfp4_add_prenorm has written (ss, `chunks` of them, eps: the norm's scale per row).  k is
// cut only into the caller's parts (consumers of few rows add them up; a gate/up matrix of so few tiles that parts would pay is small).
// w_ready: w and w_scales were written ahead of the launch that wrote these rows, and are read while it ends.
AIR_API int air_mxfp4_linear_normed(const void* packed, const void* scales, const float* ss, int chunks, float eps, const void* w, const void* w_scales,
                                    void* out, int out_dtype, int T, int N, int K, int terms, int splits, int mode, float alpha, float limit,
                                    float shift, int sms, int* status, int w_ready, cudaStream_t stream) {
    using namespace air;
    if (!mx_fits(T, K, terms) || T > 64 || N < 1 || splits < 1 || (splits > 1 && (out_dtype != AIR_F32 || mode != MX_STORE)) || sms < 2 || mode < MX_STORE ||
        mode > MX_GATED || (mode == MX_ADD && out_dtype != AIR_F32) || (mode == MX_GATED && N % 2) || !ss || chunks != (K + MXN_CHUNK - 1) / MXN_CHUNK ||
        (((uintptr_t)packed | (uintptr_t)scales | (uintptr_t)w | (uintptr_t)w_scales) & 15))
        return AIR_ERR_BAD_ARGUMENT;
    if (T == 0) return 0;
    const MxPlan p = mx_plan(T, N, K, terms, sms);
    const MxCall c{packed, scales, w, (const uint8_t*)w_scales, out, T, N, K, splits, sms, status, stream, mode, alpha, limit, shift,
                   ss, chunks, eps, w_ready};
    AIR_DISPATCH(out_dtype, TO, { return launch_mxfp4_terms<TO>(p, terms, c); });
}

AIR_API int air_trace_set_mxfp4(unsigned long long* buffer) { return air::set_trace_here(buffer); }
