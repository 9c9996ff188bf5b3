// mxfp4.hip -- microscaled 4-bit floats (gfx950): quantisation, decoding and the product of two quantised matrices.
//
// A row is cut into blocks of 32 along k.  A block holds 32 e2m1 codes (sign, magnitude 0 .5 1 1.5 2 3 4 6) and one e8m0 scale byte s
// that stands for 2^(s - 127):
//     s = max(floor(log2 max|x|) - 2, -127) + 127,      code = rne(x / 2^(s - 127)), magnitudes above 6 become 6.
// A block with an infinity or a NaN gets s = 255: all of its values read back as NaN.
//
// Layout of a matrix [M, K] (K padded with zeros to Kp = 256 c):
//     codes  [Kp / 32][M][16]      the 32 codes of (row, block) are 16 consecutive bytes, low nibble first: exactly what a lane hands to
//                                  v_mfma_scale_f32_32x32x64_f8f6f4 (lane l: row l & 31, block l >> 5), and 64 rows of one block are the
//                                  1 KB that one global -> LDS copy of a wave moves, in the order in which the fragments are read
//     scales [Kp / 256][2][M][4]   byte j of (chunk, half, row): block 8 chunk + 2 j + half.  One dword holds a lane's scales of the four
//                                  k-steps of a 256 chunk; the instruction picks the byte.
#include <type_traits>
#include "common.hpp"

namespace snf {

typedef float mx_f32x4 __attribute__((ext_vector_type(4)));
typedef float mx_f32x16 __attribute__((ext_vector_type(16)));
typedef int mx_i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(1))) const void* mx_gptr;
typedef __attribute__((address_space(3))) void* mx_lptr;

template <typename T>
struct alignas(16) MxVec {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};

__device__ __forceinline__ int mx_scale_byte(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23);  // biased exponent of the block's largest magnitude (0: zero or subnormal)
    return e == 255 ? 255 : max(e - 2, 0);
}
// 2^(byte - 127) as a float (byte < 255; byte 0 is the subnormal 2^-127)
__device__ __forceinline__ float mx_scale_float(int byte) { return __uint_as_float(byte > 0 ? (uint32_t)byte << 23 : 0x00400000u); }

// a block that is one lane's: its 16 bytes of codes and its scale byte
__device__ __forceinline__ uint4 mx_block(const float (&v)[32], int& sb) {
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    sb = mx_scale_byte(amax);
    const float sc = mx_scale_float(sb);
    uint32_t d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * i], v[8 * i + 1], sc, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * i + 2], v[8 * i + 3], sc, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * i + 4], v[8 * i + 5], sc, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[8 * i + 6], v[8 * i + 7], sc, 3);
        d[i] = sb == 255 ? 0x77777777u : c;  // (any non-zero magnitude: NaN under a NaN scale)
    }
    return make_uint4(d[0], d[1], d[2], d[3]);
}

// ---- quantisation ---------------------------------------------------------------------------------------------------------------
// A workgroup takes 32 rows x 256 columns.  A lane loads 16 bytes of a row (whole rows of the tile are contiguous), the lanes of a block
// agree on its largest magnitude by cross-lane exchanges, convert their own values and put the codes into LDS in the order of the layout;
// the tile leaves as 8 runs of 32 x 16 bytes.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void k_mxfp4_quantize(const T* __restrict__ x, int M, int K, int64_t ld, int chunks,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    constexpr int V = MxVec<T>::N, LPR = 256 / V, RPP = 256 / LPR, LPB = 32 / V;
    constexpr int KB_PITCH = 32 * 16 + 16;  // (one 16-byte column further per block: the eight blocks of a row lie in different banks)
    __shared__ __attribute__((aligned(16))) uint8_t s_codes[8 * KB_PITCH];
    __shared__ __attribute__((aligned(16))) uint8_t s_scales[2 * 32 * 4];
    const int c = (int)(blockIdx.x % (unsigned)chunks);
    const int r0 = (int)(blockIdx.x / (unsigned)chunks) * 32;
    const int lr = threadIdx.x / LPR, lc = threadIdx.x % LPR;
    const int col = c * 256 + lc * V, kb = lc / LPB, part = lc % LPB;
    float v[32 / RPP][V];
#pragma unroll
    for (int p = 0; p < 32 / RPP; ++p) {
        const int row = r0 + p * RPP + lr;
        const bool live = row < M;
        const T* src = x + (int64_t)row * ld + col;
        if (WIDE && live && col + V <= K) {
            const MxVec<T> t = *reinterpret_cast<const MxVec<T>*>(src);
#pragma unroll
            for (int i = 0; i < V; ++i) v[p][i] = (float)t.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[p][i] = live && col + i < K ? (float)src[i] : 0.f;
        }
    }
#pragma unroll
    for (int p = 0; p < 32 / RPP; ++p) {
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) amax = max(amax, __float_as_uint(v[p][i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int d = 1; d < LPB; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d, WAVE));
        const int sb = mx_scale_byte(amax);
        const float sc = mx_scale_float(sb);
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[p][0], v[p][1], sc, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[p][2], v[p][3], sc, 1);
        if constexpr (V == 8) {
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[p][4], v[p][5], sc, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[p][6], v[p][7], sc, 3);
        }
        if (sb == 255) w = 0x77777777u;  // (any non-zero magnitude: NaN under a NaN scale)
        const int lrow = p * RPP + lr;
        uint8_t* dst = s_codes + kb * KB_PITCH + lrow * 16 + part * (V / 2);
        if constexpr (V == 8) *reinterpret_cast<uint32_t*>(dst) = w;
        else *reinterpret_cast<uint16_t*>(dst) = (uint16_t)w;
        if (part == 0) s_scales[((kb & 1) * 32 + lrow) * 4 + (kb >> 1)] = (uint8_t)sb;
    }
    __syncthreads();
    {
        const int b = threadIdx.x >> 5, r = threadIdx.x & 31;
        if (r0 + r < M)
            *reinterpret_cast<uint4*>(codes + (((size_t)c * 8 + b) * M + r0 + r) * 16) =
                *reinterpret_cast<const uint4*>(s_codes + b * KB_PITCH + r * 16);
    }
    if (threadIdx.x < 64) {
        const int h = threadIdx.x >> 5, r = threadIdx.x & 31;
        if (r0 + r < M)
            reinterpret_cast<uint32_t*>(scales)[((size_t)c * 2 + h) * M + r0 + r] = reinterpret_cast<const uint32_t*>(s_scales)[h * 32 + r];
    }
}

// The operand planes of the encoder's producers (x = hi + lo, bf16, [K / 8][M][8]) instead of rows: four of their k-blocks are a block.
// A workgroup takes 64 rows x 256 k; a thread has whole blocks of one row, so nothing is exchanged but the scale bytes.
__global__ __launch_bounds__(256) void k_mxfp4_quantize_planes(const uint4* __restrict__ hi, const uint4* __restrict__ lo, int M, int K,
                                                               int chunks, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    __shared__ __attribute__((aligned(16))) uint8_t s_scales[2 * 64 * 4];
    const int c = (int)(blockIdx.x % (unsigned)chunks), lr = threadIdx.x & 63;
    const int row = (int)(blockIdx.x / (unsigned)chunks) * 64 + lr;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int b = p * 4 + (int)(threadIdx.x >> 6), kb = c * 8 + b;
        float v[32];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            uint4 h = make_uint4(0, 0, 0, 0), l = h;
            if (row < M && kb * 4 + g < K / 8) {
                h = hi[(size_t)(kb * 4 + g) * M + row];
                l = lo[(size_t)(kb * 4 + g) * M + row];
            }
            const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, lw[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[8 * g + 2 * i] = __uint_as_float(hw[i] << 16) + __uint_as_float(lw[i] << 16);
                v[8 * g + 2 * i + 1] = __uint_as_float(hw[i] & 0xFFFF0000u) + __uint_as_float(lw[i] & 0xFFFF0000u);
            }
        }
        int sb;
        const uint4 d = mx_block(v, sb);
        if (row < M) *reinterpret_cast<uint4*>(codes + ((size_t)kb * M + row) * 16) = d;
        s_scales[((b & 1) * 64 + lr) * 4 + (b >> 1)] = (uint8_t)sb;
    }
    __syncthreads();
    if (threadIdx.x < 128 && row < M)
        reinterpret_cast<uint32_t*>(scales)[((size_t)c * 2 + (threadIdx.x >> 6)) * M + row] =
            reinterpret_cast<const uint32_t*>(s_scales)[threadIdx.x];
}

// ---- decoding -------------------------------------------------------------------------------------------------------------------
// The tiles of the quantisation, the other way: codes and scales of 32 rows x 256 columns into LDS, rows out.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void k_mxfp4_dequantize(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int M,
                                                          int K, int chunks, T* __restrict__ out) {
    constexpr int V = MxVec<T>::N, LPR = 256 / V, RPP = 256 / LPR, LPB = 32 / V;
    constexpr int KB_PITCH = 32 * 16 + 16;
    __shared__ __attribute__((aligned(16))) uint8_t s_codes[8 * KB_PITCH];
    __shared__ __attribute__((aligned(16))) uint8_t s_scales[2 * 32 * 4];
    const int c = (int)(blockIdx.x % (unsigned)chunks);
    const int r0 = (int)(blockIdx.x / (unsigned)chunks) * 32;
    {
        const int b = threadIdx.x >> 5, r = threadIdx.x & 31;
        if (r0 + r < M)
            *reinterpret_cast<uint4*>(s_codes + b * KB_PITCH + r * 16) =
                *reinterpret_cast<const uint4*>(codes + (((size_t)c * 8 + b) * M + r0 + r) * 16);
    }
    if (threadIdx.x < 64) {
        const int h = threadIdx.x >> 5, r = threadIdx.x & 31;
        if (r0 + r < M)
            reinterpret_cast<uint32_t*>(s_scales)[h * 32 + r] = reinterpret_cast<const uint32_t*>(scales)[((size_t)c * 2 + h) * M + r0 + r];
    }
    __syncthreads();
    const int lr = threadIdx.x / LPR, lc = threadIdx.x % LPR;
    const int col = c * 256 + lc * V, kb = lc / LPB, part = lc % LPB;
#pragma unroll
    for (int p = 0; p < 32 / RPP; ++p) {
        const int lrow = p * RPP + lr, row = r0 + lrow;
        if (row >= M || col >= K) continue;
        const uint8_t* src = s_codes + kb * KB_PITCH + lrow * 16 + part * (V / 2);
        const uint32_t w = V == 8 ? *reinterpret_cast<const uint32_t*>(src) : (uint32_t)*reinterpret_cast<const uint16_t*>(src);
        const int sb = s_scales[((kb & 1) * 32 + lrow) * 4 + (kb >> 1)];
        const float sc = sb == 255 ? __uint_as_float(0x7FC00000u) : mx_scale_float(sb);
        MxVec<T> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            // magnitudes: codes 0, 1 are 0 and 1/2, the others (1 + m / 2) 2^(e - 1)
            const uint32_t q = (w >> (4 * i)) & 15u, e = (q >> 1) & 3u, m = q & 1u;
            const float mag = e == 0 ? 0.5f * (float)m : __uint_as_float(((e + 126u) << 23) | (m << 22));
            o.v[i] = (T)((q & 8u ? -mag : mag) * sc);
        }
        T* dst = out + (int64_t)row * K + col;
        if (WIDE && col + V <= K) {
            __builtin_nontemporal_store(__builtin_bit_cast(mx_f32x4, o), reinterpret_cast<mx_f32x4*>(dst));  // (84 MB: 17.2 us; through the caches 20.2)
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (col + i < K) dst[i] = o.v[i];
        }
    }
}

// ---- product --------------------------------------------------------------------------------------------------------------------
// nn.GELU (erf form) as max(v, 0) - |v| / 2 erfc(|v| / sqrt 2): nothing cancels.  erfc(x) = e^(-x^2) P(t), t = 1 / (1 + 0.38 x), P a
// polynomial of degree 9 without a constant, fitted to e^(x^2) erfc(x) on 0 .. 10 by reweighted least squares (relative error 2e-8);
// in fp32 the result is within 2.4e-7 of the exact one (1 + erff: 4.5e-7, and the epilogue of 4096 x 1280 -> 5120 takes 20 us longer).
__device__ __forceinline__ float mx_gelu(float v) {
    const float a = fminf(fabsf(v), 20.f), x = a * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.38f, x, 1.f));
    float q = 0.0589650683f;
    q = fmaf(q, t, -0.262271076f);
    q = fmaf(q, t, 0.36383757f);
    q = fmaf(q, t, -0.161427662f);
    q = fmaf(q, t, 0.229999989f);
    q = fmaf(q, t, 0.138662234f);
    q = fmaf(q, t, 0.203903109f);
    q = fmaf(q, t, 0.213919863f);
    q = fmaf(q, t, 0.214410931f);
    const float e = __builtin_amdgcn_exp2f(x * x * -1.4426950408889634f);
    return __builtin_elementwise_maximum(v, 0.f) - 0.5f * a * (q * t * e);
}

template <int ACT>
__device__ __forceinline__ float mx_act(float v) {
    if constexpr (ACT == SNF_ACT_RELU) return v > 0.f || v != v ? v : 0.f;
    else if constexpr (ACT == SNF_ACT_SIGMOID) return 1.f / (1.f + expf(-v));
    else if constexpr (ACT == SNF_ACT_GELU) return mx_gelu(v);
    else return v;
}
// f with the activation as a constant: one copy of an epilogue each, no branch per element
template <typename F>
__device__ __forceinline__ void mx_with_act(int act, F f) {
    switch (act) {
        case SNF_ACT_RELU: f(std::integral_constant<int, SNF_ACT_RELU>{}); break;
        case SNF_ACT_SIGMOID: f(std::integral_constant<int, SNF_ACT_SIGMOID>{}); break;
        case SNF_ACT_GELU: f(std::integral_constant<int, SNF_ACT_GELU>{}); break;
        default: f(std::integral_constant<int, SNF_ACT_NONE>{});
    }
}

constexpr int MX_PITCH = 64 + 4;  // floats of a row of the outgoing tile in LDS
constexpr int mx_stage(int bm, int bn) { return (8 * 16 + 2 * 4) * (bm + bn); }

// y[m][n] = act(sum_k a[m][k] w[n][k] + bias[n]), fp32 sums on v_mfma_scale_f32_32x32x64_f8f6f4 (products of codes are exact).
// A workgroup of WM x WN waves takes BM rows x BN columns; a stage is 256 k of both operands and their scales in LDS, two stage buffers:
// the copies of the next stage are under way during the products of this one.  The weights are the instruction's first operand: a lane
// ends up with four consecutive columns of one row, and the tile leaves through LDS in whole rows of 64 columns, where the bias and the
// activation are applied; its stores do not stay in the caches (they are half of a wide layer's time: 4900 x 1280 -> 3840 fp32 36 us with
// ordinary stores, 32 with these).
// Measured (medians): 4900 x 1280 -> 3840 fp32 (75 MB out) 32 us = 1.5 PFLOP/s, 2.3 TB/s of stores: stores, copies and products a third each;
// 16384 x 5120 -> 5120 bf16 227 us = 3.8 PFLOP/s: a tile's 256 k take 1.9 us, its products alone 1.3, its copies through L2 alone 1.0.
template <int BM, int BN, int WM, int WN, typename T>
__global__ __launch_bounds__(64 * WM * WN) void k_mxfp4_linear(const uint8_t* __restrict__ a, const uint8_t* __restrict__ as,
                                                               const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                               const float* __restrict__ bias, int M, int N, int chunks, int act,
                                                               T* __restrict__ y, uint8_t* __restrict__ y_scales, int row_tiles,
                                                               int col_tiles) {
    constexpr int WAVES = WM * WN, RB = BM / WM / 32, CB = BN / WN / 32;  // 32-row / 32-column blocks of a wave
    // a stage: codes of the rows [8][BM][16], of the columns [8][BN][16], scales of the rows [2][BM][4], of the columns [2][BN][4]
    constexpr int W_AT = 8 * BM * 16, SA_AT = W_AT + 8 * BN * 16, SW_AT = SA_AT + 8 * BM, STAGE = mx_stage(BM, BN);
    constexpr int A_PIECES = BM / 8 / WAVES, W_PIECES = BN / 8 / WAVES;  // 1 KB copies of a wave a stage: 64 rows of one block
    constexpr int S_PIECES = (BM + BN) / 32 / WAVES;                     // 256-byte copies: 64 rows' scales of one half
    constexpr int PITCH = MX_PITCH;
    static_assert(CB % 2 == 0 && A_PIECES * WAVES * 8 == BM && W_PIECES * WAVES * 8 == BN && S_PIECES * WAVES * 32 == BM + BN, "tile");
    extern __shared__ __attribute__((aligned(16))) uint8_t mx_lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, half = lane >> 5, wr = wave / WN, wc = wave % WN;
    // an XCD takes consecutive tiles, and those go down 8 row tiles before they step to the next column tile: the workgroups that run
    // together on it work on an 8 x 8 square of tiles, whose operands its L2 holds
    const int total = row_tiles * col_tiles, per = (total + 7) >> 3;
    const int slot = (int)blockIdx.x >> 3, t = ((int)blockIdx.x & 7) * per + slot;
    if (slot >= per || t >= total) return;
    const int group = t / (8 * col_tiles), in_group = t - group * 8 * col_tiles, tall = min(8, row_tiles - group * 8);
    const int rt = group * 8 + in_group % tall, ct = in_group / tall;
    const int m0 = rt * BM, n0 = ct * BN;

    mx_f32x16 acc[RB][CB];
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int j = 0; j < CB; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    // rows past the end read the last row (their results are not stored).  A wave copies the same 64 rows of every block it has: one
    // 32-bit offset a lane (M, N < 2^28) on top of addresses that are the wave's
    static_assert(WAVES % (BM / 64) == 0 && WAVES % (BN / 64) == 0, "a wave's rows");
    const uint32_t off_a = (uint32_t)min(m0 + wave % (BM / 64) * 64 + lane, M - 1) * 16u;
    const uint32_t off_w = (uint32_t)min(n0 + wave % (BN / 64) * 64 + lane, N - 1) * 16u;
    constexpr int PIECES = A_PIECES + W_PIECES + S_PIECES;
    auto copy = [&](int p, int c, uint8_t* __restrict__ stage) {  // (p is a constant where this is called)
        if (p < A_PIECES) {
            const int piece = p * WAVES + wave;
            const uint8_t* block = a + ((size_t)c * 8 + piece / (BM / 64)) * M * 16;
            __builtin_amdgcn_global_load_lds((mx_gptr)(block + off_a), (mx_lptr)(stage + piece * 1024), 16, 0, 0);
        } else if (p < A_PIECES + W_PIECES) {
            const int piece = (p - A_PIECES) * WAVES + wave;
            const uint8_t* block = w + ((size_t)c * 8 + piece / (BN / 64)) * N * 16;
            __builtin_amdgcn_global_load_lds((mx_gptr)(block + off_w), (mx_lptr)(stage + W_AT + piece * 1024), 16, 0, 0);
        } else {
            const int piece = (p - A_PIECES - W_PIECES) * WAVES + wave;  // rows' first
            const bool rows = piece < BM / 32;
            const int at = rows ? piece : piece - BM / 32, h = at / ((rows ? BM : BN) / 64), g = at % ((rows ? BM : BN) / 64);
            const int count = rows ? M : N;
            const uint8_t* scales = (rows ? as : ws) + ((size_t)c * 2 + h) * count * 4;
            __builtin_amdgcn_global_load_lds((mx_gptr)(scales + (uint32_t)min((rows ? m0 : n0) + g * 64 + lane, count - 1) * 4u),
                                             (mx_lptr)(stage + SA_AT + piece * 256), 4, 0, 0);
        }
    };
    // One stage: its products and, between them, the copies of stage c + 1 into the other buffer -- one at a time, since a copy holds its
    // wave up for some 100 cycles: all of them at the start of a stage leave the matrix cores idle that long (both waves of a SIMD issue
    // theirs at once).  (The pointers are restricted so that the reads of one buffer are known not to wait for the copies into the other.)
    auto step = [&](const uint8_t* __restrict__ from, uint8_t* __restrict__ into, int c, auto more) {
        const uint8_t* fa = from + (half * BM + wr * RB * 32 + li) * 16;
        const uint8_t* fw = from + W_AT + (half * BN + wc * CB * 32 + li) * 16;
        int sa[RB], sw[CB];
#pragma unroll
        for (int i = 0; i < RB; ++i) sa[i] = *reinterpret_cast<const int*>(from + SA_AT + (half * BM + (wr * RB + i) * 32 + li) * 4);
#pragma unroll
        for (int j = 0; j < CB; ++j) sw[j] = *reinterpret_cast<const int*>(from + SW_AT + (half * BN + (wc * CB + j) * 32 + li) * 4);
        // fragments a step ahead of their products; the scale's byte is part of the instruction
        mx_i32x8 xa[2][RB], xw[2][CB];
        auto fetch = [&](int s, mx_i32x8 (&ra)[RB], mx_i32x8 (&rw)[CB]) {
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int4 q = *reinterpret_cast<const int4*>(fa + (s * 2 * BM + i * 32) * 16);
                ra[i] = mx_i32x8{q.x, q.y, q.z, q.w, 0, 0, 0, 0};
            }
#pragma unroll
            for (int j = 0; j < CB; ++j) {
                const int4 q = *reinterpret_cast<const int4*>(fw + (s * 2 * BN + j * 32) * 16);
                rw[j] = mx_i32x8{q.x, q.y, q.z, q.w, 0, 0, 0, 0};
            }
        };
        fetch(0, xa[0], xw[0]);
#define MX_STEP(S_)                                                                                                              \
    {                                                                                                                            \
        __builtin_amdgcn_sched_barrier(0);                                                                                       \
        if ((S_) < 3) fetch((S_) + 1, xa[((S_) + 1) & 1], xw[((S_) + 1) & 1]);                                                   \
        __builtin_amdgcn_sched_barrier(0);                                                                                       \
        constexpr int LO = (S_) * PIECES / 4, HI = ((S_) + 1) * PIECES / 4;                                                      \
        _Pragma("unroll") for (int i = 0; i < RB; ++i) _Pragma("unroll") for (int j = 0; j < CB; ++j) {                          \
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(xw[(S_) & 1][j], xa[(S_) & 1][i], acc[i][j], 4, 4, S_,   \
                                                                        sw[j], S_, sa[i]);                                       \
            if constexpr (decltype(more)::value) {                                                                               \
                _Pragma("unroll") for (int p = LO; p < HI; ++p) if ((p - LO) * RB * CB / (HI - LO) == i * CB + j) {              \
                    __builtin_amdgcn_sched_barrier(0);                                                                           \
                    copy(p, c + 1, into);                                                                                        \
                    __builtin_amdgcn_sched_barrier(0);                                                                           \
                }                                                                                                                \
            }                                                                                                                    \
        }                                                                                                                        \
    }
        MX_STEP(0)
        MX_STEP(1)
        MX_STEP(2)
        MX_STEP(3)
#undef MX_STEP
        __builtin_amdgcn_sched_barrier(0);  // (the wait for the copies belongs behind the products)
        if constexpr (decltype(more)::value) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    uint8_t *const even = mx_lds, *const odd = mx_lds + STAGE;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) copy(p, 0, even);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int c = 0; c + 1 < chunks; ++c) step(c & 1 ? odd : even, c & 1 ? even : odd, c, std::true_type{});
    step((chunks - 1) & 1 ? odd : even, (chunks - 1) & 1 ? even : odd, chunks - 1, std::false_type{});
    // out, 32 rows x 64 columns at a time through the wave's own piece of LDS.  Element e of a lane: column 8 (e / 4) + 4 half + e % 4 of
    // its 32-column block, row li.
    float* out = reinterpret_cast<float*>(mx_lds) + wave * 32 * PITCH;
    constexpr bool CODES = sizeof(T) == 1;
    constexpr int V = CODES ? 32 : MxVec<T>::N, LPR = 64 / V, RPP = 64 / LPR;  // columns a lane stores at once; lanes of a row; rows of a pass
    const bool wide = N % V == 0;
    mx_with_act(act, [&](auto fixed) {
#pragma unroll
        for (int j2 = 0; j2 < CB / 2; ++j2) {
            // (codes: a lane has a block of a row; neighbouring lanes have neighbouring rows, whose blocks are neighbours in memory)
            const int nb = n0 + (wc * CB + 2 * j2) * 32, col = (CODES ? half : lane % LPR) * V;
            float b[V];
#pragma unroll
            for (int e = 0; e < V; ++e) b[e] = bias && nb + col + e < N ? bias[nb + col + e] : 0.f;
#pragma unroll
            for (int i = 0; i < RB; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const mx_f32x16& v = acc[i][2 * j2 + j];
                        *reinterpret_cast<mx_f32x4*>(out + li * PITCH + 32 * j + 8 * g + 4 * half) =
                            mx_f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                    }
                __builtin_amdgcn_wave_barrier();
                const int mb = m0 + (wr * RB + i) * 32;
                if constexpr (CODES) {  // (N is a multiple of 256)
                    float v[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) v[e] = mx_act<decltype(fixed)::value>(out[li * PITCH + col + e] + b[e]);
                    int sb;
                    const uint4 d = mx_block(v, sb);
                    const int m = mb + li, kb = (nb + col) >> 5;
                    if (m < M && nb < N) {
                        *reinterpret_cast<uint4*>(y + ((size_t)kb * M + m) * 16) = d;
                        y_scales[(((size_t)(kb >> 3) * 2 + (kb & 1)) * M + m) * 4 + ((kb & 7) >> 1)] = (uint8_t)sb;
                    }
                } else {
#pragma unroll
                    for (int p = 0; p < 32 / RPP; ++p) {
                        const int row = p * RPP + lane / LPR;
                        MxVec<T> o;
#pragma unroll
                        for (int e = 0; e < V; ++e) o.v[e] = (T)mx_act<decltype(fixed)::value>(out[row * PITCH + col + e] + b[e]);
                        if (mb + row >= M || nb + col >= N) continue;
                        T* dst = y + (int64_t)(mb + row) * N + nb + col;
                        if (wide) {
                            __builtin_nontemporal_store(__builtin_bit_cast(mx_f32x4, o), reinterpret_cast<mx_f32x4*>(dst));
                        } else {
#pragma unroll
                            for (int e = 0; e < V; ++e)
                                if (nb + col + e < N) dst[e] = o.v[e];
                        }
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
    });
}

// The same product where tiles of 128 x 128 would leave most of the chip idle: few rows (down to a single token), or few of both.  A
// workgroup takes 16 columns x 16 MT rows and its eight waves deal out the k-steps of 128 among them (v_mfma_scale_f32_16x16x128_f8f6f4);
// operands go straight from memory to registers -- a lane's 16 bytes are one block -- and the waves' sums are joined in LDS in a fixed
// order.  What bounds it is the latency of a few loads one behind the other: 1 x 1280 -> 5120 takes 5.0 us (3.5 MB of weights: 0.5 us).
// SRC: the element type of x, quantised by the lane that feeds it to the instruction (a block's 32 values are one lane's; MT = 1 only, as
// every column tile does it again), or uint8_t for codes.
template <typename SRC, int MT, bool WIDE, typename T>
__global__ __launch_bounds__(512) void k_mxfp4_linear_split(const SRC* __restrict__ x, const uint8_t* __restrict__ xs, int64_t ld,
                                                            const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws,
                                                            const float* __restrict__ bias, int M, int K, int N, int units, int act,
                                                            T* __restrict__ y, int col_tiles) {
    constexpr bool CODES = sizeof(SRC) == 1;
    static_assert(CODES || MT == 1, "rows are quantised on the way for one row tile only");
    __shared__ mx_f32x4 s_part[8][MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int n0 = (int)(blockIdx.x % (unsigned)col_tiles) * 16, m0 = (int)(blockIdx.x / (unsigned)col_tiles) * 16 * MT;
    const int n = min(n0 + r, N - 1);
    mx_f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = mx_f32x4{0.f, 0.f, 0.f, 0.f};
    // block 4 u + q of a row: byte (2 (u & 1) + q / 2) of the dword of (chunk u / 2, half q & 1)
    auto scale = [&](const uint8_t* p, int rows, int row, int u) {
        return (int)(reinterpret_cast<const uint32_t*>(p)[((size_t)(u >> 1) * 2 + (q & 1)) * rows + row] >> (16 * (u & 1) + 8 * (q >> 1)));
    };
#pragma unroll 2
    for (int u = wave; u < units; u += 8) {
        const int4 wq = *reinterpret_cast<const int4*>(w + (((size_t)u * 4 + q) * N + n) * 16);
        const int sw = scale(ws, N, n, u);
        const mx_i32x8 xw = {wq.x, wq.y, wq.z, wq.w, 0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            int4 xq = make_int4(0, 0, 0, 0);
            int sx = 0;
            if constexpr (CODES) {
                const int m = min(m0 + 16 * t + r, M - 1);
                xq = *reinterpret_cast<const int4*>(x + (((size_t)u * 4 + q) * M + m) * 16);
                sx = scale(xs, M, m, u);
            } else if (m0 + r < M) {
                constexpr int V = MxVec<SRC>::N;
                const int col = (u * 4 + q) * 32;
                const SRC* src = x + (int64_t)(m0 + r) * ld + col;
                float v[32];
#pragma unroll
                for (int g = 0; g < 32 / V; ++g) {
                    if (WIDE && col + (g + 1) * V <= K) {
                        const MxVec<SRC> c = *reinterpret_cast<const MxVec<SRC>*>(src + g * V);
#pragma unroll
                        for (int i = 0; i < V; ++i) v[g * V + i] = (float)c.v[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < V; ++i) v[g * V + i] = col + g * V + i < K ? (float)src[g * V + i] : 0.f;
                    }
                }
                const uint4 d = mx_block(v, sx);
                xq = make_int4((int)d.x, (int)d.y, (int)d.z, (int)d.w);
            }
            const mx_i32x8 xx = {xq.x, xq.y, xq.z, xq.w, 0, 0, 0, 0};
            acc[t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(xw, xx, acc[t], 4, 4, 0, sw, 0, sx);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) s_part[wave][t][lane] = acc[t];
    __syncthreads();
    // element (lane, e): row lane & 15, column 4 (lane >> 4) + e
    mx_with_act(act, [&](auto fixed) {
        for (int i = threadIdx.x; i < MT * 256; i += 512) {
            const int col = i & 15, row = i >> 4;  // consecutive threads: consecutive columns
            const int m = m0 + row, nn = n0 + col;
            if (m >= M || nn >= N) continue;
            float sum = 0.f;
#pragma unroll
            for (int p = 0; p < 8; ++p) sum += s_part[p][row >> 4][(col >> 2) * 16 + (row & 15)][col & 3];
            y[(int64_t)m * N + nn] = (T)mx_act<decltype(fixed)::value>(sum + (bias ? bias[nn] : 0.f));
        }
    });
}

static bool mx_aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

template <typename T>
static int mx_quantize_t(const T* x, int M, int K, int64_t ld, uint8_t* codes, uint8_t* scales, hipStream_t st) {
    const int chunks = ceil_div(K, 256);
    const int64_t blocks = (int64_t)ceil_div(M, 32) * chunks;
    SNF_REQUIRE(blocks * 256 < ((int64_t)1 << 32), "snf_mxfp4_quantize: %d x %d is too large for one launch", M, K);
    if (mx_aligned(x, 16) && (ld * (int64_t)sizeof(T)) % 16 == 0)
        k_mxfp4_quantize<T, true><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(x, M, K, ld, chunks, codes, scales);
    else
        k_mxfp4_quantize<T, false><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(x, M, K, ld, chunks, codes, scales);
    SNF_LAUNCH_CHECK("snf_mxfp4_quantize");
    return SNF_OK;
}

template <typename T>
static int mx_dequantize_t(const uint8_t* codes, const uint8_t* scales, int M, int K, T* out, hipStream_t st) {
    const int chunks = ceil_div(K, 256);
    const int64_t blocks = (int64_t)ceil_div(M, 32) * chunks;
    SNF_REQUIRE(blocks * 256 < ((int64_t)1 << 32), "snf_mxfp4_dequantize: %d x %d is too large for one launch", M, K);
    if (mx_aligned(out, 16) && ((int64_t)K * (int64_t)sizeof(T)) % 16 == 0)
        k_mxfp4_dequantize<T, true><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(codes, scales, M, K, chunks, out);
    else
        k_mxfp4_dequantize<T, false><<<dim3((unsigned)blocks), dim3(256), 0, st>>>(codes, scales, M, K, chunks, out);
    SNF_LAUNCH_CHECK("snf_mxfp4_dequantize");
    return SNF_OK;
}

template <int BM, int BN, int WM, int WN, typename T>
static int mx_tiles(const uint8_t* a, const uint8_t* as, const uint8_t* w, const uint8_t* ws, const float* bias, int M, int N, int chunks,
                    int act, T* y, uint8_t* y_scales, hipStream_t st) {
    constexpr int THREADS = 64 * WM * WN, STAGES = 2 * mx_stage(BM, BN), OUT = WM * WN * 32 * MX_PITCH * 4, LDS = STAGES > OUT ? STAGES : OUT;
    const int rts = ceil_div(M, BM), cts = ceil_div(N, BN);
    SNF_REQUIRE(((int64_t)rts * cts + 8) * THREADS < ((int64_t)1 << 32), "snf_mxfp4_linear: %d x %d is too large for one launch", M, N);
    const auto kernel = k_mxfp4_linear<BM, BN, WM, WN, T>;
    if (LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        SNF_REQUIRE(e == hipSuccess, "snf_mxfp4_linear: %d bytes of LDS: %s", LDS, hipGetErrorString(e));
    }
    const int per = (rts * cts + 7) / 8;
    kernel<<<dim3(8 * per), dim3(THREADS), LDS, st>>>(a, as, w, ws, bias, M, N, chunks, act, y, y_scales, rts, cts);
    SNF_LAUNCH_CHECK("snf_mxfp4_linear");
    return SNF_OK;
}

template <typename T>
static int mx_tiled(const uint8_t* a, const uint8_t* as, const uint8_t* w, const uint8_t* ws, const float* bias, int M, int N, int chunks,
                    int act, T* y, uint8_t* y_scales, hipStream_t st) {
    // (bytes from the caches halve with tiles of 256 x 256, but one workgroup fills a CU and nothing runs beside its loads and stores:
    // 16384 x 5120 -> 5120 fp32 243 us against 280, 16384 x 1280 -> 5120 100 against 104, both with 1280 such tiles; with 640 and 320 of
    // them 8192 x 1280 -> 5120 takes 58 against 52, 4096 x 1280 -> 5120 40 against 32)
    if ((int64_t)ceil_div(M, 256) * ceil_div(N, 256) >= 1024)
        return mx_tiles<256, 256, 4, 2, T>(a, as, w, ws, bias, M, N, chunks, act, y, y_scales, st);
    return mx_tiles<128, 128, 2, 2, T>(a, as, w, ws, bias, M, N, chunks, act, y, y_scales, st);
}

template <typename T>
static int mx_linear_t(const uint8_t* a, const uint8_t* as, const uint8_t* w, const uint8_t* ws, const float* bias, int M, int K, int N,
                       int act, T* y, hipStream_t st) {
    const int chunks = ceil_div(K, 256);
    // (tiles of 128 x 128 walk all of k, one workgroup each: few of them leave the chip idle.  512 x 5120 -> 1280, 40 tiles: split 10.0 us,
    // tiles 18.1; 1024 x 5120 -> 1280, 80 tiles: 21.1 and 18.5; 512 x 1280 -> 5120, 160 tiles: 13.4 and 9.8)
    if ((int64_t)ceil_div(M, 128) * ceil_div(N, 128) < 64) {
        const int cts = ceil_div(N, 16), mt = M <= 16 ? 1 : M <= 32 ? 2 : 4, rts = ceil_div(M, 16 * mt);
        SNF_REQUIRE((int64_t)rts * cts * 512 < ((int64_t)1 << 32), "snf_mxfp4_linear: %d x %d is too large for one launch", M, N);
        const dim3 grid((unsigned)(rts * cts)), block(512);
        if (mt == 1) k_mxfp4_linear_split<uint8_t, 1, true, T><<<grid, block, 0, st>>>(a, as, 0, w, ws, bias, M, K, N, 2 * chunks, act, y, cts);
        else if (mt == 2) k_mxfp4_linear_split<uint8_t, 2, true, T><<<grid, block, 0, st>>>(a, as, 0, w, ws, bias, M, K, N, 2 * chunks, act, y, cts);
        else k_mxfp4_linear_split<uint8_t, 4, true, T><<<grid, block, 0, st>>>(a, as, 0, w, ws, bias, M, K, N, 2 * chunks, act, y, cts);
        SNF_LAUNCH_CHECK("snf_mxfp4_linear (split)");
        return SNF_OK;
    }
    return mx_tiled(a, as, w, ws, bias, M, N, chunks, act, y, (uint8_t*)nullptr, st);
}

template <typename SRC, typename T>
static int mx_rows_t(const SRC* x, int64_t ld, const uint8_t* w, const uint8_t* ws, const float* bias, int M, int K, int N, int act, T* y,
                     hipStream_t st) {
    const int cts = ceil_div(N, 16), units = 2 * ceil_div(K, 256);
    if (mx_aligned(x, 16) && (ld * (int64_t)sizeof(SRC)) % 16 == 0)
        k_mxfp4_linear_split<SRC, 1, true, T><<<dim3(cts), dim3(512), 0, st>>>(x, nullptr, ld, w, ws, bias, M, K, N, units, act, y, cts);
    else
        k_mxfp4_linear_split<SRC, 1, false, T><<<dim3(cts), dim3(512), 0, st>>>(x, nullptr, ld, w, ws, bias, M, K, N, units, act, y, cts);
    SNF_LAUNCH_CHECK("snf_mxfp4_linear_rows");
    return SNF_OK;
}

template <typename SRC>
static int mx_rows_src(const SRC* x, int64_t ld, const uint8_t* w, const uint8_t* ws, const float* bias, int M, int K, int N, int act,
                       void* y, int out_dtype, hipStream_t st) {
    switch (out_dtype) {
        case SNF_F32: return mx_rows_t(x, ld, w, ws, bias, M, K, N, act, (float*)y, st);
        case SNF_BF16: return mx_rows_t(x, ld, w, ws, bias, M, K, N, act, (__bf16*)y, st);
        case SNF_F16: return mx_rows_t(x, ld, w, ws, bias, M, K, N, act, (_Float16*)y, st);
    }
    SNF_REQUIRE(false, "snf_mxfp4_linear_rows: unknown dtype %d", out_dtype);
}

}  // namespace snf

extern "C" {

int snf_mxfp4_quantize(const void* x, int dtype, int M, int K, int64_t ld, uint8_t* codes, uint8_t* scales, snf_stream_t stream) {
    SNF_REQUIRE(M >= 0 && K >= 1, "snf_mxfp4_quantize: bad sizes M=%d K=%d", M, K);
    if (M == 0) return SNF_OK;
    SNF_REQUIRE(x && codes && scales, "snf_mxfp4_quantize: null pointer");
    SNF_REQUIRE(ld >= K || M == 1, "snf_mxfp4_quantize: rows of %d values overlap at stride %lld", K, (long long)ld);
    SNF_REQUIRE(snf::mx_aligned(codes, 16) && snf::mx_aligned(scales, 4), "snf_mxfp4_quantize: codes / scales are not aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case SNF_F32: return snf::mx_quantize_t((const float*)x, M, K, ld, codes, scales, st);
        case SNF_BF16: return snf::mx_quantize_t((const __bf16*)x, M, K, ld, codes, scales, st);
        case SNF_F16: return snf::mx_quantize_t((const _Float16*)x, M, K, ld, codes, scales, st);
    }
    SNF_REQUIRE(false, "snf_mxfp4_quantize: unknown dtype %d", dtype);
}

int snf_mxfp4_quantize_planes(const uint16_t* hi, const uint16_t* lo, int M, int K, uint8_t* codes, uint8_t* scales, snf_stream_t stream) {
    SNF_REQUIRE(M >= 0 && K >= 8 && K % 8 == 0, "snf_mxfp4_quantize_planes: bad sizes M=%d K=%d", M, K);
    if (M == 0) return SNF_OK;
    SNF_REQUIRE(hi && lo && codes && scales, "snf_mxfp4_quantize_planes: null pointer");
    SNF_REQUIRE(snf::mx_aligned(hi, 16) && snf::mx_aligned(lo, 16) && snf::mx_aligned(codes, 16) && snf::mx_aligned(scales, 4),
                "snf_mxfp4_quantize_planes: an operand is not aligned");
    const int chunks = snf::ceil_div(K, 256);
    const int64_t blocks = (int64_t)snf::ceil_div(M, 64) * chunks;
    SNF_REQUIRE(blocks * 256 < ((int64_t)1 << 32), "snf_mxfp4_quantize_planes: %d x %d is too large for one launch", M, K);
    snf::k_mxfp4_quantize_planes<<<dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream>>>((const uint4*)hi, (const uint4*)lo, M, K, chunks,
                                                                                               codes, scales);
    SNF_LAUNCH_CHECK("snf_mxfp4_quantize_planes");
    return SNF_OK;
}

int snf_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int M, int K, void* out, int dtype, snf_stream_t stream) {
    SNF_REQUIRE(M >= 0 && K >= 1, "snf_mxfp4_dequantize: bad sizes M=%d K=%d", M, K);
    if (M == 0) return SNF_OK;
    SNF_REQUIRE(out && codes && scales, "snf_mxfp4_dequantize: null pointer");
    SNF_REQUIRE(snf::mx_aligned(codes, 16) && snf::mx_aligned(scales, 4), "snf_mxfp4_dequantize: codes / scales are not aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case SNF_F32: return snf::mx_dequantize_t(codes, scales, M, K, (float*)out, st);
        case SNF_BF16: return snf::mx_dequantize_t(codes, scales, M, K, (__bf16*)out, st);
        case SNF_F16: return snf::mx_dequantize_t(codes, scales, M, K, (_Float16*)out, st);
    }
    SNF_REQUIRE(false, "snf_mxfp4_dequantize: unknown dtype %d", dtype);
}

int snf_mxfp4_linear(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* w_codes, const uint8_t* w_scales, const float* bias,
                     int M, int K, int N, int act, void* y, int dtype, snf_stream_t stream) {
    SNF_REQUIRE(M >= 0 && K >= 1 && N >= 1, "snf_mxfp4_linear: bad sizes M=%d K=%d N=%d", M, K, N);
    SNF_REQUIRE(M < 1 << 28 && N < 1 << 28, "snf_mxfp4_linear: M=%d, N=%d are 2^28 at most", M, N);
    SNF_REQUIRE(act >= SNF_ACT_NONE && act <= SNF_ACT_GELU, "snf_mxfp4_linear: unknown activation %d", act);
    if (M == 0) return SNF_OK;
    SNF_REQUIRE(a_codes && a_scales && w_codes && w_scales && y, "snf_mxfp4_linear: null pointer");
    SNF_REQUIRE(snf::mx_aligned(a_codes, 16) && snf::mx_aligned(w_codes, 16) && snf::mx_aligned(a_scales, 4) && snf::mx_aligned(w_scales, 4) &&
                    snf::mx_aligned(y, 16),
                "snf_mxfp4_linear: an operand is not aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case SNF_F32: return snf::mx_linear_t(a_codes, a_scales, w_codes, w_scales, bias, M, K, N, act, (float*)y, st);
        case SNF_BF16: return snf::mx_linear_t(a_codes, a_scales, w_codes, w_scales, bias, M, K, N, act, (__bf16*)y, st);
        case SNF_F16: return snf::mx_linear_t(a_codes, a_scales, w_codes, w_scales, bias, M, K, N, act, (_Float16*)y, st);
    }
    SNF_REQUIRE(false, "snf_mxfp4_linear: unknown dtype %d", dtype);
}

int snf_mxfp4_linear_quantized(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* w_codes, const uint8_t* w_scales,
                               const float* bias, int M, int K, int N, int act, uint8_t* y_codes, uint8_t* y_scales, snf_stream_t stream) {
    SNF_REQUIRE(M >= 0 && K >= 1 && N >= 256 && N % 256 == 0, "snf_mxfp4_linear_quantized: bad sizes M=%d K=%d N=%d", M, K, N);
    SNF_REQUIRE(M < 1 << 28 && N < 1 << 28, "snf_mxfp4_linear_quantized: M=%d, N=%d are 2^28 at most", M, N);
    SNF_REQUIRE(act >= SNF_ACT_NONE && act <= SNF_ACT_GELU, "snf_mxfp4_linear_quantized: unknown activation %d", act);
    if (M == 0) return SNF_OK;
    SNF_REQUIRE(a_codes && a_scales && w_codes && w_scales && y_codes && y_scales, "snf_mxfp4_linear_quantized: null pointer");
    SNF_REQUIRE(snf::mx_aligned(a_codes, 16) && snf::mx_aligned(w_codes, 16) && snf::mx_aligned(a_scales, 4) && snf::mx_aligned(w_scales, 4) &&
                    snf::mx_aligned(y_codes, 16) && snf::mx_aligned(y_scales, 4),
                "snf_mxfp4_linear_quantized: an operand is not aligned");
    return snf::mx_tiled(a_codes, a_scales, w_codes, w_scales, bias, M, N, snf::ceil_div(K, 256), act, y_codes, y_scales, (hipStream_t)stream);
}

int snf_mxfp4_linear_rows(const void* x, int dtype, int64_t ld, const uint8_t* w_codes, const uint8_t* w_scales, const float* bias, int M,
                          int K, int N, int act, void* y, int out_dtype, snf_stream_t stream) {
    SNF_REQUIRE(M >= 0 && M <= SNF_MXFP4_ROWS && K >= 1 && N >= 1, "snf_mxfp4_linear_rows: bad sizes M=%d K=%d N=%d", M, K, N);
    SNF_REQUIRE(act >= SNF_ACT_NONE && act <= SNF_ACT_GELU, "snf_mxfp4_linear_rows: unknown activation %d", act);
    if (M == 0) return SNF_OK;
    SNF_REQUIRE(x && w_codes && w_scales && y, "snf_mxfp4_linear_rows: null pointer");
    SNF_REQUIRE(ld >= K || M == 1, "snf_mxfp4_linear_rows: rows of %d values overlap at stride %lld", K, (long long)ld);
    SNF_REQUIRE(snf::mx_aligned(w_codes, 16) && snf::mx_aligned(w_scales, 4), "snf_mxfp4_linear_rows: an operand is not aligned");
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case SNF_F32: return snf::mx_rows_src((const float*)x, ld, w_codes, w_scales, bias, M, K, N, act, y, out_dtype, st);
        case SNF_BF16: return snf::mx_rows_src((const __bf16*)x, ld, w_codes, w_scales, bias, M, K, N, act, y, out_dtype, st);
        case SNF_F16: return snf::mx_rows_src((const _Float16*)x, ld, w_codes, w_scales, bias, M, K, N, act, y, out_dtype, st);
    }
    SNF_REQUIRE(false, "snf_mxfp4_linear_rows: unknown dtype %d", dtype);
}

}  // extern "C"
