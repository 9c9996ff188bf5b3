// distill.hip -- a teacher's top logits and the distillation loss that reads them (gfx950).
//   snf_top_logits     : the k largest logits of a row in order, and log sum exp(x / T) over all the others
//   snf_top_distill_*  : T^2 KL(teacher || student) per row, from the teacher's top logits (and the mass of the rest, as one class of its
//                        own), with the student's gradient
// Bound by reading the rows: a part of a row stays in registers (16 bytes a load, all under way at once) while its maximum and its sum of
// exponentials are taken; rows may begin at any element of a 16-byte granule.  4096 rows of 65536 bf16, k = 64 (medians): selection 142 us
// (streaming 94 us = 5.7 TB/s, then 48), loss 166 us (reading 144 us = 3.7 TB/s, then 17 + 5), gradient 179 us (1.07 GB, 6.0 TB/s).
#include "common.hpp"

namespace snf {

constexpr int TD_MAX_K = 256;
constexpr float TD_LOG2E = 1.4426950408889634f;
constexpr float TD_NINF = -INFINITY;

template <typename T>
__device__ __forceinline__ void td_unpack(const uint4& r, float (&f)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void td_unpack<float>(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
}
template <>
__device__ __forceinline__ void td_unpack<__bf16>(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <>
__device__ __forceinline__ void td_unpack<_Float16>(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] & 0xFFFFu));
        f[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
    }
}
// -inf in element e of a packed register set
template <typename T>
__device__ __forceinline__ void td_clear(uint4& r, int e) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    if constexpr (sizeof(T) == 4) {
        w[e] = 0xFF800000u;
    } else {
        const uint32_t ninf = __is_same(T, __bf16) ? 0xFF80u : 0xFC00u;
        w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xFFFFu) | ninf << 16 : (w[e >> 1] & 0xFFFF0000u) | ninf;
    }
}

// order of the logits as unsigned numbers: -0 is 0, a NaN is above everything
__device__ __forceinline__ uint32_t td_key(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const uint32_t b = x == 0.f ? 0u : __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float td_value(uint32_t key) {
    if (key == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
    return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ float td_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // a NaN stays
__device__ __forceinline__ float td_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// exp((x - m) / T), c = log2(e) / T; nothing is left of x = -inf, also where the maximum is.  x - m, c and their product are rounded to
// 32 bits: off by up to 3 |x - m| / T 2^-24 of itself, which a sum does not feel (what lies far below the maximum is little of it).
__device__ __forceinline__ float td_term(float x, float m, float c) { return x == TD_NINF ? 0.f : td_exp2((x - m) * c); }

// The same where each value counts by itself (a gradient's entry far below the maximum, a sum's factor): what the three roundings leave
// out is carried along and multiplied on, so that the result is off by 5 steps of 2^-24 however far x lies below m.
struct TdScale {
    float c, low;  // log2(e) / T in two parts
    __device__ __forceinline__ explicit TdScale(float temperature) {
        constexpr float log2e_low = (float)(1.4426950408889634 - (double)TD_LOG2E);
        c = TD_LOG2E / temperature;
        low = (fmaf(-c, temperature, TD_LOG2E) + log2e_low) / temperature;
    }
    __device__ __forceinline__ float exp(float x, float m) const {  // (x = -inf: 0, where m is finite)
        const float d = x - m, back = x - d, lost = (x - (d + back)) + (back - m);
        const float t = d * c, rest = fmaf(lost, c, fmaf(d, low, fmaf(d, c, -t)));
        return td_exp2(t) * __builtin_amdgcn_fmed3f(fmaf(rest, 0.69314718f, 1.f), 0.5f, 2.f);  // (rest is NaN where d is infinite)
    }
    __device__ __forceinline__ float term(float x, float m) const { return x == TD_NINF ? 0.f : exp(x, m); }
};

struct TdMaxOp { __device__ static float op(float a, float b) { return td_max(a, b); } };
struct TdSumOp { __device__ static float op(float a, float b) { return a + b; } };
struct TdCountOp { __device__ static int op(int a, int b) { return a + b; } };

template <int CTRL, typename V>
__device__ __forceinline__ V td_dpp(V v) {
    return __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
// over 8 neighbouring lanes / over the wave, in every lane, without LDS: lane swaps inside a quad, mirrored halves and rows of 16 lanes,
// then rows and halves of the wave exchanged
template <typename OP, typename V>
__device__ __forceinline__ V td_reduce8(V v) {
    v = OP::op(v, td_dpp<0xB1>(v));   // quad: 1 0 3 2
    v = OP::op(v, td_dpp<0x4E>(v));   // quad: 2 3 0 1
    return OP::op(v, td_dpp<0x141>(v));  // 8 lanes mirrored
}
template <typename OP, typename V>
__device__ __forceinline__ V td_reduce_wave(V v) {
    v = td_reduce8<OP>(v);
    v = OP::op(v, td_dpp<0x140>(v));  // 16 lanes mirrored
    const unsigned a = __builtin_bit_cast(unsigned, v);
    const auto r16 = __builtin_amdgcn_permlane16_swap(a, a, false, false);
    v = OP::op(__builtin_bit_cast(V, (unsigned)r16[0]), __builtin_bit_cast(V, (unsigned)r16[1]));
    const unsigned b = __builtin_bit_cast(unsigned, v);
    const auto r32 = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return OP::op(__builtin_bit_cast(V, (unsigned)r32[0]), __builtin_bit_cast(V, (unsigned)r32[1]));
}
// the same value in every thread of the workgroup; `s` is scratch of one word per wave, free again after the call
template <int THREADS, typename OP, typename V>
__device__ __forceinline__ V td_reduce(V v, V* s) {
    v = td_reduce_wave<OP>(v);
    if constexpr (THREADS > WAVE) {
        if (lane_id() == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[0];
#pragma unroll
        for (int i = 1; i < THREADS / WAVE; ++i) v = OP::op(v, s[i]);
        __syncthreads();
    }
    return v;
}

// A part [p0, p0 + len) of a row in the registers of a workgroup.  Loads are whole 16-byte granules of memory: the first one may begin
// `shift` elements before the part and the last one end behind it; what does not belong to the part is -inf.
template <typename T, int THREADS, int NV>
struct TdPart {
    static constexpr int E = 16 / (int)sizeof(T);
    uint4 r[NV];
    int shift, len;

    __device__ __forceinline__ void load(const T* p, int n) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        shift = (int)((a & 15) / sizeof(T));
        len = n;
        const uint4* g = reinterpret_cast<const uint4*>(a & ~(uintptr_t)15);
        const int granules = (shift + n + E - 1) / E;
        constexpr uint32_t fill = __is_same(T, float) ? 0xFF800000u : __is_same(T, __bf16) ? 0xFF80FF80u : 0xFC00FC00u;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int v = j * THREADS + (int)threadIdx.x;
            r[j] = make_uint4(fill, fill, fill, fill);
            if (v < granules) r[j] = g[v];
        }
        // the granules at the two ends
        const int last = granules - 1;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int v = j * THREADS + (int)threadIdx.x;
            if (v == 0 || v == last) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!inside(place(j, e))) td_clear<T>(r[j], e);
            }
        }
    }
    __device__ __forceinline__ int place(int j, int e) const { return (j * THREADS + (int)threadIdx.x) * E + e - shift; }
    __device__ __forceinline__ bool inside(int place) const { return (unsigned)place < (unsigned)len; }
    // (the empty asm keeps the unpacked values of one pass from staying in registers for the next)
    template <typename F>
    __device__ __forceinline__ void each(F f) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float x[E];
            asm volatile("" : "+v"(r[j].x), "+v"(r[j].y), "+v"(r[j].z), "+v"(r[j].w));
            td_unpack<T>(r[j], x);
#pragma unroll
            for (int e = 0; e < E; ++e) f(x[e], j, e);
        }
    }
};

// =================================================================================================================================
// top logits
// =================================================================================================================================
// A bound first: of G >= k disjoint sets of elements take the maxima; at least k elements reach the k-th largest of them, and few others
// do (G = 2 k sets of values in random order: about 1.4 k elements).  What reaches the bound goes to LDS as 64-bit keys (value, place: all
// different, so the order of arrival plays no part), and a key's rank is the number of larger keys.  The log-sum-exp of the rest refers to
// the largest logit of the rest, so that it keeps its digits however far below the top it lies; it is never a difference.
//   short rows (TD_SHAPES): the row in the registers of one workgroup, the sets are threads: one launch, one read.
//   long rows: k_top_groups streams them -- any number of workgroups a row, nothing exchanged between waves -- and leaves the maximum and
//     the sum of exponentials of every 128 bytes; k_top_select, one workgroup a row, finds the bound among the maxima and reads again only
//     the groups that reach it (about 1.4 k of them: 9 % of a row of 65536 bf16 at k = 64; the groups' results are 6 %).
// Rows with a NaN and rows where more than TD_CAND elements reach the bound (long runs of equal logits, sorted rows) take the exact way,
// from memory (td_select_exact).
constexpr int TD_CAND = 1024;
constexpr int TD_GROUP = 8;  // 16-byte granules of a group (td_reduce8)

template <int THREADS>
struct TdSelect {
    static constexpr int CAND = THREADS == 64 ? 256 : TD_CAND;
    alignas(16) uint64_t key[CAND + 8];  // (filled up with zeros to a multiple of 8: a zero is below every key)
    uint64_t sorted[CAND];
    alignas(16) float set[THREADS];
    float red[THREADS / WAVE];
    uint32_t bound;
    int n;
};

// the k-th largest of the sets' maxima; a set is THREADS / sets neighbouring threads (a power of two, at most 16), none has a NaN
template <int THREADS>
__device__ __forceinline__ float td_bound(TdSelect<THREADS>& s, float own, int k, int sets) {
    const int per = THREADS / sets;
    if (per >= 2) own = td_max(own, td_dpp<0xB1>(own));
    if (per >= 4) own = td_max(own, td_dpp<0x4E>(own));
    if (per >= 8) own = td_max(own, td_dpp<0x141>(own));
    if (per >= 16) own = td_max(own, td_dpp<0x140>(own));
    if ((int)threadIdx.x % per == 0) s.set[threadIdx.x / per] = own;
    __syncthreads();
    if ((int)threadIdx.x < sets) {
        const float mine = s.set[threadIdx.x];
        int ge = 0;
#pragma unroll 8
        for (int i = 0; i < sets / 4; ++i) {
            const float4 f = reinterpret_cast<const float4*>(s.set)[i];
            ge += (f.x >= mine) + (f.y >= mine) + (f.z >= mine) + (f.w >= mine);
        }
        if (ge >= k) atomicMax(&s.bound, td_key(mine));
    }
    __syncthreads();
    return td_value(s.bound);
}

// keys of s.n <= CAND candidates in order; the first k leave
template <int THREADS, typename T>
__device__ __forceinline__ void td_rank(TdSelect<THREADS>& s, int k, int32_t* __restrict__ ids, T* __restrict__ logits) {
    const int n = s.n;
    if (threadIdx.x < 8) s.key[n + threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t mine = s.key[i];
        int rank = 0;
        for (int j = 0; j < n; j += 8) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(s.key + j + 2 * q);
                rank += (two.x > mine) + (two.y > mine);
            }
        }
        s.sorted[rank] = mine;
        if (rank < k) {
            ids[rank] = (int32_t)~(uint32_t)mine;
            logits[rank] = (T)td_value((uint32_t)(mine >> 32));
        }
    }
    __syncthreads();
}

__device__ __forceinline__ float td_lse(float m, float sum, float temperature) {
    return m == INFINITY || m == TD_NINF ? m : m / temperature + logf(sum);
}

// elements of a row from memory, in the order of their places: all of them, or those of the listed groups (in rising order)
template <typename T>
struct TdSlots {
    static constexpr int E = 16 / (int)sizeof(T);
    const uint4* g;
    const int* list;
    int shift, V, granules, slots;
    __device__ __forceinline__ TdSlots(const T* p, int V_, const int* list_, int listed) : list(list_), V(V_) {
        shift = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
        g = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)15);
        granules = (shift + V + E - 1) / E;
        slots = list ? listed * TD_GROUP : granules;
    }
    template <typename F>
    __device__ __forceinline__ void one(int slot, F f) const {
        const int v = list ? list[slot / TD_GROUP] * TD_GROUP + slot % TD_GROUP : slot;
        if (v >= granules) return;
        float x[E];
        td_unpack<T>(g[v], x);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int at = v * E + e - shift;
            if ((unsigned)at < (unsigned)V) f(x[e], at);
        }
    }
    template <int THREADS, typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
        for (int slot = (int)threadIdx.x; slot < slots; slot += THREADS) one(slot, f);
    }
};

// The exact way.  `in` holds every element whose key is at least `from` (0: not known), at least k of them; groups whose maximum is below
// `bound` are in `stats` instead where that is given.  The k-th key is `from` itself where fewer than k lie above it (long runs of equal
// logits: a few passes over `in`; 4096 rows of 65536 equal bf16, k = 64: 0.90 ms, 4.70 by bisection), else found by bisection of its bits
// (the same rows ascending: 0.57 ms over the listed groups, 4.57 over all; with a NaN, over all: 3.3 ms); equals of the k-th are taken in
// the order of their places, which ends as soon as there are enough.  Leaves the k keys in s (for td_rank), returns the rest's log-sum-exp.
template <typename T, int THREADS>
__device__ __noinline__ float td_select_exact(TdSelect<THREADS>& s, const TdSlots<T> in, uint32_t from, const float2* stats, int groups,
                                              float bound, int k, float temperature) {
    const float c = TD_LOG2E / temperature;
    int* red = reinterpret_cast<int*>(s.red);
    auto count = [&](auto pred) {
        int n = 0;
        in.template each<THREADS>([&](float v, int) { n += pred(td_key(v)); });
        return td_reduce<THREADS, TdCountOp>(n, red);
    };
    uint32_t kth = from;
    int above = from ? count([&](uint32_t key) { return key > from; }) : k;
    if (above >= k) {
        kth = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t t = kth | 1u << bit;
            if (count([&](uint32_t key) { return key >= t; }) >= k) kth = t;
        }
        above = count([&](uint32_t key) { return key > kth; });
    }
    const int need = k - above, equal = count([&](uint32_t key) { return key == kth; });
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    float m = equal > need ? td_value(kth) : TD_NINF, sum = 0.f;
    in.template each<THREADS>([&](float v, int p) {
        const uint32_t key = td_key(v);
        if (key > kth) s.key[atomicAdd(&s.n, 1)] = (uint64_t)key << 32 | (uint32_t)~p;
        else if (key < kth) m = td_max(m, v);
    });
    int taken = 0;
    for (int base = 0; base < in.slots && taken < need; base += THREADS) {
        const int slot = base + (int)threadIdx.x;
        int mine = 0;
        if (slot < in.slots) in.one(slot, [&](float v, int) { mine += td_key(v) == kth; });
        int incl = mine;
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const int t = __shfl_up(incl, d, WAVE);
            if (lane_id() >= d) incl += t;
        }
        if (lane_id() == WAVE - 1) red[threadIdx.x >> 6] = incl;
        __syncthreads();
        int at = taken + incl - mine;
#pragma unroll 1
        for (int w = 0; w < THREADS / WAVE; ++w) {
            at += w < (int)(threadIdx.x >> 6) ? red[w] : 0;
            taken += red[w];
        }
        __syncthreads();
        if (mine && at < need)
            in.one(slot, [&](float v, int p) {
                if (td_key(v) == kth && at++ < need) s.key[atomicAdd(&s.n, 1)] = (uint64_t)kth << 32 | (uint32_t)~p;
            });
    }
    __syncthreads();
    auto others = [&](auto f) {
        if (stats)
            for (int i = threadIdx.x; i < groups; i += THREADS)
                if (stats[i].x < bound) f(stats[i]);
    };
    others([&](float2 st) { m = td_max(m, st.x); });
    m = td_reduce<THREADS, TdMaxOp>(m, s.red);
    others([&](float2 st) { sum += st.y * td_term(st.x, m, c); });
    in.template each<THREADS>([&](float v, int) { if (td_key(v) < kth) sum += td_term(v, m, c); });
    sum = td_reduce<THREADS, TdSumOp>(sum, s.red);
    if (equal > need) sum += (float)(equal - need) * td_term(td_value(kth), m, c);  // (else kth may be far above m)
    return td_lse(m, sum, temperature);
}

template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void k_top_logits(const T* __restrict__ x, int V, int64_t ld, int k, int sets, float temperature,
                                                        int32_t* __restrict__ ids, T* __restrict__ logits, float* __restrict__ rest) {
    using Sel = TdSelect<THREADS>;
    __shared__ Sel s;
    const int64_t row = blockIdx.x;
    ids += row * k;
    logits += row * k;
    const T* src = x + row * ld;
    TdPart<T, THREADS, NV> reg;
    reg.load(src, V);
    const float c = TD_LOG2E / temperature;
    if (threadIdx.x == 0) { s.bound = 0; s.n = 0; }
    float own = TD_NINF;
    reg.each([&](float v, int, int) { own = td_max(own, v); });
    const float top = td_reduce<THREADS, TdMaxOp>(own, s.red);
    float bound = 0.f;
    bool exact = top != top;
    if (!exact) {
        bound = td_bound<THREADS>(s, own, k, sets);
        if (own >= bound)
            reg.each([&](float v, int j, int e) {
                if (v >= bound) {
                    const int p = reg.place(j, e);
                    if (reg.inside(p)) {
                        const int at = atomicAdd(&s.n, 1);
                        if (at < Sel::CAND) s.key[at] = (uint64_t)td_key(v) << 32 | (uint32_t)~p;
                    }
                }
            });
        __syncthreads();
        exact = s.n > Sel::CAND;
    }
    if (exact) {
        const float r = td_select_exact<T, THREADS>(s, TdSlots<T>(src, V, nullptr, 0), top != top ? 0u : td_key(bound), nullptr, 0, bound, k,
                                                    temperature);
        td_rank<THREADS>(s, k, ids, logits);
        if (threadIdx.x == 0) rest[row] = r;
        return;
    }
    td_rank<THREADS>(s, k, ids, logits);
    const int n = s.n;
    float m, sum = 0.f;
    if (n > k) {
        m = td_value((uint32_t)(s.sorted[k] >> 32));
    } else {
        m = TD_NINF;
        reg.each([&](float v, int, int) { if (v < bound) m = td_max(m, v); });
        m = td_reduce<THREADS, TdMaxOp>(m, s.red);
    }
    if (m > TD_NINF) reg.each([&](float v, int, int) { sum += v < bound ? td_exp2((v - m) * c) : 0.f; });
    for (int i = k + threadIdx.x; i < n; i += THREADS) sum += td_term(td_value((uint32_t)(s.sorted[i] >> 32)), m, c);
    sum = td_reduce<THREADS, TdSumOp>(sum, s.red);
    if (threadIdx.x == 0) rest[row] = td_lse(m, sum, temperature);
}

// maximum and sum of exp((x - maximum) / T) of every group of TD_GROUP granules; a lane holds one granule of NV groups
template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void k_top_groups(const T* __restrict__ x, int V, int64_t ld, float temperature, int chunks, int groups,
                                                        float2* __restrict__ out) {
    constexpr int E = 16 / (int)sizeof(T);
    const int64_t row = blockIdx.x / (unsigned)chunks;
    const int g0 = (int)(blockIdx.x % (unsigned)chunks) * (THREADS * NV);  // the first granule
    const T* src = x + row * ld;
    const int shift = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    const uint4* g = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15);
    const int last = (shift + V + E - 1) / E - 1;
    const float c = TD_LOG2E / temperature;
    uint4 r[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) r[j] = g[min(g0 + j * THREADS + (int)threadIdx.x, last)];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int v = g0 + j * THREADS + (int)threadIdx.x;
        float f[E];
        td_unpack<T>(r[j], f);
        if (v == 0 || v >= last) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if ((unsigned)(v * E + e - shift) >= (unsigned)V) f[e] = TD_NINF;
        }
        float m = f[0];
#pragma unroll
        for (int e = 1; e < E; ++e) m = td_max(m, f[e]);
        m = td_reduce8<TdMaxOp>(m);
        const float ref = m == TD_NINF ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += td_exp2((f[e] - ref) * c);
        sum = td_reduce8<TdSumOp>(sum);
        if (v % TD_GROUP == 0 && v <= last) out[row * groups + v / TD_GROUP] = make_float2(m, sum);
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void k_top_select(const T* __restrict__ x, int V, int64_t ld, int k, int sets, float temperature, int groups,
                                                        const float2* __restrict__ stats, int32_t* __restrict__ ids, T* __restrict__ logits,
                                                        float* __restrict__ rest) {
    using Sel = TdSelect<THREADS>;
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ Sel s;
    __shared__ int s_list[TD_CAND];  // the groups that reach the bound, in an order of their own (the sums below are always the same sums)
    __shared__ int s_count[THREADS / WAVE];
    const int64_t row = blockIdx.x;
    ids += row * k;
    logits += row * k;
    stats += row * groups;
    const T* src = x + row * ld;
    const int shift = (int)((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    const uint4* g = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(src) & ~(uintptr_t)15);
    const int granules = (shift + V + E - 1) / E, live = (granules + TD_GROUP - 1) / TD_GROUP;
    const float c = TD_LOG2E / temperature;
    if (threadIdx.x == 0) { s.bound = 0; s.n = 0; }
    // a thread's first four groups, and later its first four granules of the groups that are read again, stay in registers
    constexpr int KEEP = 4;
    float2 kept[KEEP];
#pragma unroll
    for (int q = 0; q < KEEP; ++q) {
        const int i = q * THREADS + (int)threadIdx.x;
        kept[q] = i < live ? stats[i] : make_float2(TD_NINF, 0.f);
    }
    auto each_group = [&](auto f) {
#pragma unroll
        for (int q = 0; q < KEEP; ++q) {
            const int i = q * THREADS + (int)threadIdx.x;
            if (i < live) f(kept[q], i);
        }
        for (int i = KEEP * THREADS + (int)threadIdx.x; i < live; i += THREADS) f(stats[i], i);
    };
    float own = TD_NINF;
    each_group([&](float2 st, int) { own = td_max(own, st.x); });
    const float top = td_reduce<THREADS, TdMaxOp>(own, s.red);
    bool exact = top != top;
    float bound = 0.f, m = TD_NINF;  // m: the largest element below the bound
    int found = 0;
    if (!exact) {
        bound = td_bound<THREADS>(s, own, k, sets);
        int hits = 0;
        each_group([&](float2 st, int) {
            if (st.x >= bound) ++hits;
            else m = td_max(m, st.x);
        });
        int incl = hits;
#pragma unroll
        for (int d = 1; d < WAVE; d <<= 1) {
            const int t = __shfl_up(incl, d, WAVE);
            if (lane_id() >= d) incl += t;
        }
        if (lane_id() == WAVE - 1) s_count[threadIdx.x >> 6] = incl;
        __syncthreads();
        int at = incl - hits;
#pragma unroll
        for (int w = 0; w < THREADS / WAVE; ++w) {
            at += w < (int)(threadIdx.x >> 6) ? s_count[w] : 0;
            found += s_count[w];
        }
        if (hits && found <= TD_CAND)
            each_group([&](float2 st, int i) { if (st.x >= bound) s_list[at++] = i; });
        __syncthreads();
        exact = found > TD_CAND;
    }
    const int team = (int)threadIdx.x / TD_GROUP, member = (int)threadIdx.x % TD_GROUP;
    uint4 again[KEEP];
    if (!exact) {
#pragma unroll
        for (int q = 0; q < KEEP; ++q) {
            const int l = q * (THREADS / TD_GROUP) + team;
            if (l < found) again[q] = g[min(s_list[l] * TD_GROUP + member, granules - 1)];
        }
    }
    auto sweep = [&](auto f) {
        auto one = [&](const uint4& r, int l) {
            const int v = s_list[l] * TD_GROUP + member;
            float x_[E];
            td_unpack<T>(r, x_);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if ((unsigned)(v * E + e - shift) < (unsigned)V) f(x_[e], v * E + e - shift);
        };
#pragma unroll
        for (int q = 0; q < KEEP; ++q) {
            const int l = q * (THREADS / TD_GROUP) + team;
            if (l < found) one(again[q], l);
        }
        for (int l = KEEP * (THREADS / TD_GROUP) + team; l < found; l += THREADS / TD_GROUP)
            one(g[min(s_list[l] * TD_GROUP + member, granules - 1)], l);
    };
    if (!exact) {
        sweep([&](float v, int p) {
            if (v >= bound) {
                const int at = atomicAdd(&s.n, 1);
                if (at < Sel::CAND) s.key[at] = (uint64_t)td_key(v) << 32 | (uint32_t)~p;
            } else {
                m = td_max(m, v);
            }
        });
        __syncthreads();
        exact = s.n > Sel::CAND;
    }
    if (exact) {
        const bool listed = top == top && found <= TD_CAND;
        if (listed) {  // in rising order
            int* order = reinterpret_cast<int*>(s.sorted);
            for (int i = threadIdx.x; i < found; i += THREADS) {
                int rank = 0;
                for (int j = 0; j < found; ++j) rank += s_list[j] < s_list[i];
                order[rank] = s_list[i];
            }
            __syncthreads();
            for (int i = threadIdx.x; i < found; i += THREADS) s_list[i] = order[i];
            __syncthreads();
        }
        const float r = td_select_exact<T, THREADS>(s, TdSlots<T>(src, V, listed ? s_list : nullptr, found), top != top ? 0u : td_key(bound),
                                                    listed ? stats : nullptr, live, bound, k, temperature);
        td_rank<THREADS>(s, k, ids, logits);
        if (threadIdx.x == 0) rest[row] = r;
        return;
    }
    td_rank<THREADS>(s, k, ids, logits);
    const int n = s.n;
    m = td_reduce<THREADS, TdMaxOp>(m, s.red);
    if (n > k) m = td_value((uint32_t)(s.sorted[k] >> 32));
    float sum = 0.f;
    if (m > TD_NINF) {
        each_group([&](float2 st, int) { if (st.x < bound) sum += st.y * td_term(st.x, m, c); });
        sweep([&](float v, int) { if (v < bound) sum += td_term(v, m, c); });
    }
    for (int i = k + threadIdx.x; i < n; i += THREADS) sum += td_term(td_value((uint32_t)(s.sorted[i] >> 32)), m, c);
    sum = td_reduce<THREADS, TdSumOp>(sum, s.red);
    if (threadIdx.x == 0) rest[row] = td_lse(m, sum, temperature);
}

// =================================================================================================================================
// distillation loss
// =================================================================================================================================
// z [V] a student's logits, ids / t [K] the teacher's top logits (a negative id: no entry), optionally r = log sum exp(t_v / T) over all
// other places.  p = softmax over (t / T [, r]), q = softmax(z / T), q_rest = the sum of q over the places that ids does not name:
//     loss = T^2 [ sum_k p_k (log p_k - log q_{id_k}) + p_rest (log p_rest - log q_rest) ]
//     dloss / dz_v = T [ q_v - sum_{k: id_k = v} p_k - (v not named) p_rest q_v / q_rest ]
// Both are differences of numbers that are mostly alike once a student follows its teacher, and where the list holds little of the mass, or
// one place nearly all of it, also before: sums of p (log p - log q), 1 - p_rest / q_rest and q - p then have no digits left.  So the sums
// over the named and the other places are taken apart, and
//   the loss is T^2 sum over the entries and the rest of p (log p - log q) + q - p      (- the q of places that are named once more: they
//     count once): the additions cancel over all classes, every term is at least 0, an error of the logarithms counts by p - q alone;
//   with r, P and Q the named places' mass over the rest's on either side and x = (Q - P) / (1 + P):
//     log p_rest - log q_rest = log1p(x),     q_v - p_rest q_v / q_rest = -x q_v;
//   at a named place that holds more than half of both masses, q - p is the other places' p less their q.
// 100000 places, k = 8, T = 4, rows whose divergence is 7e-4: the loss is off by 2e-6 of itself, the other places' gradient by 4e-7 (by
// 4.5e-3 and 8e-5 as the plain sum of p (log p - log q) and as 1 - p_rest / q_rest).
// What the backward pass needs of a row (12 + 4 K bytes): the reference m_r and the factor f with dz_v = gs f exp((z_v - m_r) / T) for all
// places that are not named, and q - p of the named ones.
__device__ __forceinline__ float td_load(const void* p, int dtype, int64_t i) {
    if (dtype == SNF_F32) return reinterpret_cast<const float*>(p)[i];
    if (dtype == SNF_BF16) return (float)reinterpret_cast<const __bf16*>(p)[i];
    return (float)reinterpret_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ int64_t td_id(const void* ids, int wide, int64_t i) {
    return wide ? reinterpret_cast<const int64_t*>(ids)[i] : (int64_t)reinterpret_cast<const int32_t*>(ids)[i];
}

struct TdTeacher {
    const void* ids;
    const void* logits;
    const float* rest;
    int ids_wide, dtype, K;
};
struct TdSaved {
    float* rows;     // [R] loss of a row, times weight T^2; 0 where there is no target
    float* counted;  // [R] 1 or 0
    float2* stats;   // [R] m_r, f
    float* diff;     // [R, K] q - p of a named place at the first entry that names it, 0 at others
};

// p (log p - log q) + q - p with d = log p - log q, at least 0; near d = 0, where the three cancel, p (d^2 / 2 - d^3 / 6 + ...), whose first
// term left out is 2e-9 of the sum at |d| = 1/2
__device__ __forceinline__ float td_divergence(float p, float q, float d) {
    if (p == 0.f) return q;
    if (!(fabsf(d) <= 0.5f)) return p * d + (q - p);
    float c = -1.f / 362880.f;
    c = fmaf(c, d, 1.f / 40320.f);
    c = fmaf(c, d, -1.f / 5040.f);
    c = fmaf(c, d, 1.f / 720.f);
    c = fmaf(c, d, -1.f / 120.f);
    c = fmaf(c, d, 1.f / 24.f);
    c = fmaf(c, d, -1.f / 6.f);
    c = fmaf(c, d, 0.5f);
    return p * (d * d * c);
}

// One wave: the row's teacher side and its loss, from the student's maximum and sum over the places that are not named.
template <typename T>
__device__ __forceinline__ void td_finish_row(const T* __restrict__ zrow, int V, int64_t row, const TdTeacher& t, float temperature,
                                              float scale, float m_r, float s_r, const TdSaved& out) {
    constexpr int Q = TD_MAX_K / WAVE;
    const int lane = lane_id();
    const TdScale by_t(temperature);
    const bool with_rest = t.rest != nullptr;
    // (the rest is a logarithm of what has been divided by T; without it the difference is taken first)
    const float before = with_rest ? temperature : 1.f, after = with_rest ? 1.f : temperature;
    int id[Q];
    float tv[Q], zv[Q];
    bool bad = false, any = false;
    float tm = TD_NINF, nm = TD_NINF;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int k = q * WAVE + lane;
        id[q] = -1;
        tv[q] = zv[q] = TD_NINF;
        if (k < t.K) {
            const int64_t i = td_id(t.ids, t.ids_wide, row * t.K + k);
            bad |= i >= V;
            if (i >= 0 && i < V) {
                id[q] = (int)i;
                any = true;
                zv[q] = (float)zrow[i];
                nm = td_max(nm, zv[q]);
                tv[q] = td_load(t.logits, t.dtype, row * t.K + k) / before;
                tm = td_max(tm, tv[q]);
            }
        }
    }
    bad = __any(bad);
    any = __any(any) || bad;
    tm = td_reduce_wave<TdMaxOp>(tm);
    const float r = with_rest ? t.rest[row] : TD_NINF;
    if (with_rest) tm = td_max(tm, r);
    if (!any || (tm == TD_NINF && !bad)) {  // no target: no entry, or a teacher without any mass
        if (lane == 0) {
            out.rows[row] = 0.f;
            out.counted[row] = 0.f;
            out.stats[row] = make_float2(0.f, 0.f);
        }
        for (int k = lane; k < t.K; k += WAVE) out.diff[row * t.K + k] = 0.f;
        return;
    }
    // teacher: exponentials, their sum
    float pe[Q], ps = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        tv[q] = (tv[q] - tm) / after;
        pe[q] = id[q] >= 0 ? expf(tv[q]) : 0.f;
        ps += pe[q];
    }
    const float pn = td_reduce_wave<TdSumOp>(ps);
    const float re = with_rest ? expf(r - tm) : 0.f;
    ps = pn + re;
    // student: the named places, each once (and the mass of those that are named again)
    nm = td_reduce_wave<TdMaxOp>(nm);
    const float m = td_max(m_r, nm);
    float en[Q], sn = 0.f, again = 0.f;
    bool first[Q], twice = false;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        en[q] = 0.f;
        first[q] = false;
        if (q * WAVE >= t.K) continue;
        uint64_t named = 0;  // lanes whose place an earlier entry names
#pragma unroll
        for (int q2 = 0; q2 <= q; ++q2)
            for (int l0 = 0; l0 < WAVE && q2 * WAVE + l0 < t.K; l0 += 8) {
#pragma unroll
                for (int l = l0; l < l0 + 8; ++l) {
                    const uint64_t same = __ballot(id[q] == __builtin_amdgcn_readlane(id[q2], l));
                    named |= q2 < q ? same : same & (~1ull << l);
                }
            }
        first[q] = id[q] >= 0 && !(named >> lane & 1);
        if (id[q] >= 0) {
            en[q] = by_t.term(zv[q], m);
            if (first[q]) sn += en[q];
            else again += en[q];
            twice |= !first[q];
        }
    }
    sn = td_reduce_wave<TdSumOp>(sn);
    const float rest_scale = by_t.term(m_r, m), su = s_r * rest_scale, s = sn + su;
    // loss
    const float log_ps = logf(ps), log_s = logf(s);
    float loss = -again / s;
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (id[q] >= 0) loss += td_divergence(pe[q] / ps, en[q] / s, (tv[q] - log_ps) - ((zv[q] - m) / temperature - log_s));
    loss = td_reduce_wave<TdSumOp>(loss);
    const float pr = re / ps, P = pn / re, x = (sn / su - P) / (1.f + P);  // (x is not finite where one of the rests has no mass)
    const bool near = fabsf(x) <= 0.5f;
    const float d = near ? log1pf(x) : (r - tm - log_ps) - ((m_r - m) / temperature + logf(s_r) - log_s);
    loss += td_divergence(pr, su / s, d);
    // gradient
    float ref = m_r, f = near ? -x * rest_scale / s : rest_scale / s - (pr == 0.f ? 0.f : pr / s_r);
    if (m_r == TD_NINF) { ref = 0.f; f = 0.f; }  // every place is named, or what is not is -inf
    float pv[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) pv[q] = pe[q];
    if (__any(twice)) {
#pragma unroll
        for (int q2 = 0; q2 < Q; ++q2)
            for (int l = 0; l < WAVE; ++l) {
                if (q2 * WAVE + l >= t.K) break;
                const int other = __builtin_amdgcn_readlane(id[q2], l);
                const float mass = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pe[q2]), l));
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    if (other == id[q] && (q2 != q || l != lane)) pv[q] += mass;
            }
    }
    int heavy = -1;  // the named place with more than half of both masses, if there is one
#pragma unroll
    for (int q = 0; q < Q; ++q)
        if (first[q] && en[q] > 0.5f * s && pv[q] > 0.5f * ps) heavy = id[q];
    const uint64_t found = __ballot(heavy >= 0);
    float heavy_diff = 0.f;
    if (found) {
        heavy = __builtin_amdgcn_readlane(heavy, __builtin_ctzll(found));
        float po = 0.f, qo = 0.f;
#pragma unroll
        for (int q = 0; q < Q; ++q)
            if (id[q] != heavy) {
                po += pe[q];
                if (first[q]) qo += en[q];
            }
        po = td_reduce_wave<TdSumOp>(po) + re;
        qo = td_reduce_wave<TdSumOp>(qo) + su;
        heavy_diff = po / ps - qo / s;
    }
    if (bad) loss = f = __uint_as_float(0x7FC00000u);  // an id past the end
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int k = q * WAVE + lane;
        const float diff = !first[q] ? 0.f : id[q] == heavy ? heavy_diff : en[q] / s - pv[q] / ps;
        if (k < t.K) out.diff[row * t.K + k] = bad ? f : diff;
    }
    if (lane == 0) {
        out.rows[row] = loss * scale;
        out.counted[row] = 1.f;
        out.stats[row] = make_float2(ref, f);
    }
}

template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void k_top_distill_rows(const T* __restrict__ z, int V, int64_t ld, TdTeacher t, float temperature,
                                                              float scale, int parts, int part_len, TdSaved out,
                                                              float2* __restrict__ part_ms) {
    using Part = TdPart<T, THREADS, NV>;
    constexpr int WORDS = (THREADS * NV * Part::E + 31) / 32;
    __shared__ uint32_t s_named[WORDS];
    __shared__ float s_red[THREADS / WAVE];
    const int64_t row = blockIdx.x / (unsigned)parts;
    const int part = (int)(blockIdx.x % (unsigned)parts);
    const int p0 = part * part_len, len = min(part_len, V - p0);
    const T* zrow = z + row * ld;
    // (the ids are asked for before the row: loads come back in order)
    int64_t first_id = -1;
    if ((int)threadIdx.x < t.K) first_id = td_id(t.ids, t.ids_wide, row * t.K + threadIdx.x);
    Part reg;
    reg.load(zrow + p0, len);
    // the named places become -inf: one bit per place of the part, in the order of the registers
    for (int i = threadIdx.x; i < WORDS; i += THREADS) s_named[i] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < t.K; k += THREADS) {
        const int64_t i = (k < THREADS ? first_id : td_id(t.ids, t.ids_wide, row * t.K + k)) - p0;
        if (i >= 0 && i < len) atomicOr(&s_named[(i + reg.shift) >> 5], 1u << ((i + reg.shift) & 31));
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int b = (j * THREADS + (int)threadIdx.x) * Part::E;
        const uint32_t bits = s_named[b >> 5] >> (b & 31) & ((1u << Part::E) - 1u);
        if (bits)
#pragma unroll
            for (int e = 0; e < Part::E; ++e)
                if (bits >> e & 1u) td_clear<T>(reg.r[j], e);
    }
    const float c = TD_LOG2E / temperature;
    float m = TD_NINF, s = 0.f;
    reg.each([&](float v, int, int) { m = td_max(m, v); });
    m = td_reduce<THREADS, TdMaxOp>(m, s_red);
    if (m != TD_NINF) reg.each([&](float v, int, int) { s += td_exp2((v - m) * c); });
    s = td_reduce<THREADS, TdSumOp>(s, s_red);
    if (parts > 1) {
        if (threadIdx.x == 0) part_ms[row * parts + part] = make_float2(m, s);
    } else if (threadIdx.x < WAVE) {
        td_finish_row<T>(zrow, V, row, t, temperature, scale, m, s, out);
    }
}

// rows in parts: the parts' maxima and sums joined, then the row as above; one wave per row
template <typename T>
__global__ __launch_bounds__(64) void k_top_distill_join(const T* __restrict__ z, int V, int64_t ld, TdTeacher t, float temperature,
                                                         float scale, int parts, TdSaved out, const float2* __restrict__ part_ms) {
    const int64_t row = blockIdx.x;
    const float c = TD_LOG2E / temperature;
    float m = TD_NINF, s = 0.f;
    for (int p = lane_id(); p < parts; p += WAVE) m = td_max(m, part_ms[row * parts + p].x);
    m = td_reduce_wave<TdMaxOp>(m);
    for (int p = lane_id(); p < parts; p += WAVE) {
        const float2 ms = part_ms[row * parts + p];
        s += ms.y * td_term(ms.x, m, c);
    }
    s = td_reduce_wave<TdSumOp>(s);
    td_finish_row<T>(z + row * ld, V, row, t, temperature, scale, m, s, out);
}

// the loss, and what the rows' gradients are divided by; one workgroup, sums in a fixed order
__global__ __launch_bounds__(1024) void k_top_distill_mean(const float* __restrict__ rows, const float* __restrict__ counted, int R,
                                                           int mean, float* __restrict__ loss, float* __restrict__ divisor) {
    __shared__ float s_red[1024 / WAVE];
    float s = 0.f, n = 0.f;
    for (int i = threadIdx.x; i < R; i += 1024) {
        s += rows[i];
        n += counted[i];
    }
    s = td_reduce<1024, TdSumOp>(s, s_red);
    n = td_reduce<1024, TdSumOp>(n, s_red);
    if (threadIdx.x == 0) {
        const float d = mean ? fmaxf(n, 1.f) : 1.f;
        loss[0] = s / d;
        divisor[0] = d;
    }
}

// dz of a chunk of a row.  PACKED: rows of z and dz begin at the same offset from a 16-byte granule, which are then moved whole except at
// the ends of the chunk and around named places.
constexpr int TD_CHUNK = 8192;

template <typename T, bool PACKED>
__global__ __launch_bounds__(256) void k_top_distill_bwd(const T* __restrict__ z, int V, int64_t ld, const void* __restrict__ ids,
                                                         int ids_wide, int K, float temperature, float scale, int chunks,
                                                         const float* __restrict__ g, int g_per_row, const float* __restrict__ divisor,
                                                         const float* __restrict__ counted, const float2* __restrict__ stats,
                                                         const float* __restrict__ diff, T* __restrict__ dz) {
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ uint32_t s_named[TD_CHUNK / 32 + 1];
    __shared__ int s_id[TD_MAX_K];
    __shared__ float s_diff[TD_MAX_K];
    constexpr int KEEP = 4;
    const int64_t row = blockIdx.x / (unsigned)chunks;
    const int p0 = (int)(blockIdx.x % (unsigned)chunks) * TD_CHUNK, len = min(TD_CHUNK, V - p0);
    const T* zp = z + row * ld + p0;
    T* dp = dz + row * V + p0;
    // what does not depend on anything is asked for first: the row's scalars, a thread's id and its q - p, its first granules
    int64_t first_id = -1;
    float first_diff = 0.f;
    if ((int)threadIdx.x < K) {
        first_id = td_id(ids, ids_wide, row * K + threadIdx.x);
        first_diff = diff[row * K + threadIdx.x];
    }
    const int shift = PACKED ? (int)((reinterpret_cast<uintptr_t>(zp) & 15) / sizeof(T)) : 0;
    const int granules = (shift + len + E - 1) / E;
    const uint4* zg = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(zp) & ~(uintptr_t)15);
    uint4 r[KEEP];
    if (PACKED) {
#pragma unroll
        for (int q = 0; q < KEEP; ++q) r[q] = zg[min((int)(q * blockDim.x + threadIdx.x), granules - 1)];
    }
    const bool live = counted[row] != 0.f;
    const float gs = g[g_per_row ? row : 0] * scale / (divisor ? divisor[0] : 1.f);
    const TdScale by_t(temperature);
    const float2 st = stats[row];
    const float f = gs * st.y;
    // (the half types round far more away than the shorter form does)
    auto gradient = [&](float x) { return (T)(f * (sizeof(T) == 4 ? by_t.exp(x, st.x) : td_exp2((x - st.x) * by_t.c))); };
    if (live) {
        for (int i = threadIdx.x; i <= (shift + len) / 32; i += blockDim.x) s_named[i] = 0;
        __syncthreads();
        for (int k = threadIdx.x; k < K; k += blockDim.x) {
            const int64_t i = (k < (int)blockDim.x ? first_id : td_id(ids, ids_wide, row * K + k)) - p0;
            const bool here = i >= 0 && i < len;
            s_id[k] = here ? (int)i : -1;
            s_diff[k] = k < (int)blockDim.x ? first_diff : diff[row * K + k];
            if (here) atomicOr(&s_named[(i + shift) >> 5], 1u << ((i + shift) & 31));
        }
        __syncthreads();
        for (int k = threadIdx.x; k < K; k += blockDim.x) {
            const int i = s_id[k];
            if (i < 0) continue;
            float sum = 0.f;
            bool first = true;
            for (int o = 0; o < K; ++o)
                if (s_id[o] == i) {
                    first &= o >= k;
                    sum += s_diff[o];  // (not 0 once at most)
                }
            if (first) dp[i] = (T)(gs * sum);
        }
    }
    if constexpr (PACKED) {
        uint4* dg = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(dp) & ~(uintptr_t)15);
        for (int v0 = 0; v0 < granules; v0 += KEEP * blockDim.x) {
            if (v0 > 0) {
#pragma unroll
                for (int q = 0; q < KEEP; ++q) r[q] = zg[min((int)(v0 + q * blockDim.x + threadIdx.x), granules - 1)];
            }
#pragma unroll
            for (int q = 0; q < KEEP; ++q) {
                const int v = v0 + q * blockDim.x + threadIdx.x, b = v * E;
                if (v >= granules) continue;
                float x[E];
                struct alignas(16) { T v[E]; } o;
                td_unpack<T>(r[q], x);
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = live ? gradient(x[e]) : (T)0.f;
                const uint32_t bits = live ? s_named[b >> 5] >> (b & 31) & ((1u << E) - 1u) : 0u;
                if (bits == 0 && b >= shift && b + E <= shift + len) {
                    dg[v] = *reinterpret_cast<const uint4*>(&o);
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (!(bits >> e & 1u) && b + e >= shift && b + e < shift + len) dp[b + e - shift] = o.v[e];
                }
            }
        }
    } else {
        for (int i = threadIdx.x; i < len; i += blockDim.x)
            if (!live) dp[i] = (T)0.f;
            else if (!(s_named[i >> 5] >> (i & 31) & 1u)) dp[i] = gradient((float)zp[i]);
    }
}

// ---- launch shapes ----------------------------------------------------------------------------------------------------------------
// shapes a row (or a part of it) is held in, smallest first: threads x 16-byte granules a thread
struct TdShape { int threads, nv; };
constexpr TdShape TD_SHAPES[] = {{64, 1}, {64, 4}, {64, 8}, {256, 4}, {512, 4}};
// elements of a part at any alignment of its first (a multiple of E)
constexpr int td_capacity(int shape, int E) { return TD_SHAPES[shape].threads * TD_SHAPES[shape].nv * E - E; }

struct TdPlan { int shape, parts, part_len; };

// Loss: the smallest wave that holds a row; long rows are dealt out in parts of 8 KB, a wave each (no barriers, and every wave's loads are
// under way at once: 4096 x 65536 bf16, in turn and at their best, in 150 us with workgroups of 256 threads x 16 KB, 130 with waves), of
// 4 KB where that makes fewer than 256 of them.
static TdPlan td_rows_plan(int R, int V, int E) {
    int s = 0;
    while (s < 2 && td_capacity(s, E) < V) ++s;
    if (s == 2 && (int64_t)R * ceil_div(V, td_capacity(s, E)) < 256) s = 1;
    const int parts = ceil_div(V, td_capacity(s, E));
    return {s, parts, parts == 1 ? V : td_capacity(s, E)};
}

// Selection: the smallest shape that holds a row and has 2 k threads (sets for the bound; k for k > 256 / 2 threads of the largest), or -1:
// a long row.
static int td_top_shape(int V, int k, int E) {
    if (k <= 32 && td_capacity(0, E) >= V) return 0;
    if (k <= 32 && td_capacity(1, E) >= V) return 1;
    if (k <= 128 && td_capacity(3, E) >= V) return 3;
    if (k > 128 && td_capacity(4, E) >= V) return 4;
    return -1;
}
// groups of a row, wherever it begins in a granule
static int td_top_group_count(int V, int E) { return ceil_div((int64_t)V + E - 1, E * TD_GROUP); }

template <typename T>
static int td_top_t(const T* x, int R, int V, int64_t ld, int k, float temperature, int32_t* ids, T* logits, float* rest, void* ws,
                    hipStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    const int shape = td_top_shape(V, k, E);
    const int threads = shape >= 0 ? TD_SHAPES[shape].threads : k <= 128 ? 256 : 512;
    SNF_REQUIRE((int64_t)R * threads < ((int64_t)1 << 32), "snf_top_logits: %d rows are too many for one launch", R);
    int sets = 32;
    while (sets < 2 * k) sets *= 2;
    if (sets > threads) sets = threads;
#define TD_GO(S_)                                                                                                                     \
    case S_:                                                                                                                          \
        k_top_logits<T, TD_SHAPES[S_].threads, TD_SHAPES[S_].nv><<<dim3(R), dim3(threads), 0, st>>>(x, V, ld, k, sets, temperature, ids,  \
                                                                                                    logits, rest);                    \
        break;
    if (shape >= 0) {
        switch (shape) { TD_GO(0) TD_GO(1) TD_GO(3) TD_GO(4) }
        SNF_LAUNCH_CHECK("snf_top_logits");
        return SNF_OK;
    }
#undef TD_GO
    const int groups = td_top_group_count(V, E), granules = groups * TD_GROUP;
    // 16 KB a workgroup; 4 KB where that makes fewer than 1024 of them (64 x 65536 bf16, k = 64: both kernels 17.6 us with 4 KB, 18.3 with
    // 16; from 120 such rows on, and for one row of 32000 or 10^6 fp32, within the 3 % that two runs differ by)
    const int64_t big = (int64_t)R * ceil_div(granules, 256 * 4);
    const int per = big < 1024 ? 64 * 4 : 256 * 4, chunks = ceil_div(granules, per);
    SNF_REQUIRE((int64_t)R * chunks * (per / 4) < ((int64_t)1 << 32), "snf_top_logits: %d rows of %d are too many for one launch", R, V);
    const dim3 grid((unsigned)((int64_t)R * chunks));
    if (per == 256) k_top_groups<T, 64, 4><<<grid, dim3(64), 0, st>>>(x, V, ld, temperature, chunks, groups, (float2*)ws);
    else k_top_groups<T, 256, 4><<<grid, dim3(256), 0, st>>>(x, V, ld, temperature, chunks, groups, (float2*)ws);
    SNF_LAUNCH_CHECK("snf_top_logits (groups)");
    if (threads == 256) k_top_select<T, 256><<<dim3(R), dim3(256), 0, st>>>(x, V, ld, k, sets, temperature, groups, (const float2*)ws, ids, logits, rest);
    else k_top_select<T, 512><<<dim3(R), dim3(512), 0, st>>>(x, V, ld, k, sets, temperature, groups, (const float2*)ws, ids, logits, rest);
    SNF_LAUNCH_CHECK("snf_top_logits (select)");
    return SNF_OK;
}

// weight and weight T^2, which the rows' divergences are multiplied by: 0 or a normal number (weight T, the gradient's factor, is between)
static bool td_weight_ok(float weight, float temperature) {
    const double w = fabs((double)weight), scale = w * temperature * temperature;
    return weight == 0.f || (w >= FLT_MIN && w <= FLT_MAX && scale >= FLT_MIN && scale <= FLT_MAX);
}

template <typename T>
static int td_fwd_t(const T* z, int R, int V, int64_t ld, const TdTeacher& t, float temperature, float weight, const TdSaved& out, void* ws,
                    hipStream_t st) {
    const TdPlan pl = td_rows_plan(R, V, 16 / (int)sizeof(T));
    SNF_REQUIRE((int64_t)R * pl.parts * TD_SHAPES[pl.shape].threads < ((int64_t)1 << 32), "snf_top_distill_fwd: %d rows of %d are too many for one launch", R, V);
    const float scale = (float)((double)weight * temperature * temperature);
    const dim3 grid((unsigned)((int64_t)R * pl.parts));
#define TD_GO(S_)                                                                                                                     \
    case S_:                                                                                                                          \
        k_top_distill_rows<T, TD_SHAPES[S_].threads, TD_SHAPES[S_].nv><<<grid, dim3(TD_SHAPES[S_].threads), 0, st>>>(           \
            z, V, ld, t, temperature, scale, pl.parts, pl.part_len, out, (float2*)ws);                                                \
        break;
    switch (pl.shape) { TD_GO(0) TD_GO(1) TD_GO(2) }
#undef TD_GO
    SNF_LAUNCH_CHECK("snf_top_distill_fwd");
    if (pl.parts > 1) {
        k_top_distill_join<T><<<dim3(R), dim3(64), 0, st>>>(z, V, ld, t, temperature, scale, pl.parts, out, (const float2*)ws);
        SNF_LAUNCH_CHECK("snf_top_distill_fwd (join)");
    }
    return SNF_OK;
}

static int td_mean(const float* rows, const float* counted, int R, int mean, float* loss, float* divisor, hipStream_t st) {
    k_top_distill_mean<<<dim3(1), dim3(1024), 0, st>>>(rows, counted, R, mean, loss, divisor);
    SNF_LAUNCH_CHECK("snf_top_distill_fwd (mean)");
    return SNF_OK;
}

template <typename T>
static int td_bwd_t(const T* z, int R, int V, int64_t ld, const void* ids, int ids_wide, int K, float temperature, float weight,
                    const float* g, int g_per_row, const float* divisor, const float* counted, const float2* stats, const float* diff,
                    T* dz, hipStream_t st) {
    const int chunks = ceil_div(V, TD_CHUNK);
    SNF_REQUIRE((int64_t)R * chunks * 256 < ((int64_t)1 << 32), "snf_top_distill_bwd: %d rows of %d are too many for one launch", R, V);
    const dim3 grid((unsigned)((int64_t)R * chunks)), block(V <= 1024 ? 64 : 256);
    const size_t zb = ((size_t)ld * sizeof(T)) % 16, db = ((size_t)V * sizeof(T)) % 16;
    const bool packed = (R == 1 || zb == db) && (reinterpret_cast<uintptr_t>(z) & 15) == (reinterpret_cast<uintptr_t>(dz) & 15);
    if (packed)
        k_top_distill_bwd<T, true><<<grid, block, 0, st>>>(z, V, ld, ids, ids_wide, K, temperature, weight * temperature, chunks, g, g_per_row,
                                                           divisor, counted, stats, diff, dz);
    else
        k_top_distill_bwd<T, false><<<grid, block, 0, st>>>(z, V, ld, ids, ids_wide, K, temperature, weight * temperature, chunks, g,
                                                            g_per_row, divisor, counted, stats, diff, dz);
    SNF_LAUNCH_CHECK("snf_top_distill_bwd");
    return SNF_OK;
}

}  // namespace snf

extern "C" {

int64_t snf_top_logits_workspace_bytes(int R, int V, int k, int dtype) {
    if (R < 1 || V < 1 || k < 1 || k > snf::TD_MAX_K || k > V) return 0;
    const int E = dtype == SNF_F32 ? 4 : 8;
    return snf::td_top_shape(V, k, E) >= 0 ? 0 : (int64_t)R * snf::td_top_group_count(V, E) * 8;
}

int snf_top_logits(const void* x, int dtype, int R, int V, int64_t ld, int k, float temperature, int32_t* ids, void* logits, float* rest,
                   void* workspace, int64_t workspace_bytes, snf_stream_t stream) {
    SNF_REQUIRE(R >= 0 && V >= 1 && V <= SNF_TOP_MAX_V, "snf_top_logits: bad sizes R=%d V=%d", R, V);
    SNF_REQUIRE(k >= 1 && k <= snf::TD_MAX_K && k <= V, "snf_top_logits: k=%d is not in 1 .. min(V, %d)", k, snf::TD_MAX_K);
    SNF_REQUIRE(temperature >= FLT_MIN && temperature < INFINITY, "snf_top_logits: temperature %g", (double)temperature);
    SNF_REQUIRE(dtype >= SNF_F32 && dtype <= SNF_F16, "snf_top_logits: unknown dtype %d", dtype);
    if (R == 0) return SNF_OK;
    SNF_REQUIRE(x && ids && logits && rest, "snf_top_logits: null pointer");
    SNF_REQUIRE(ld >= V || R == 1, "snf_top_logits: rows of %d values overlap at stride %lld", V, (long long)ld);
    SNF_REQUIRE(workspace_bytes >= snf_top_logits_workspace_bytes(R, V, k, dtype) && (workspace_bytes == 0 || workspace),
                "snf_top_logits: workspace of %lld bytes is too small", (long long)workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case SNF_F32: return snf::td_top_t((const float*)x, R, V, ld, k, temperature, ids, (float*)logits, rest, workspace, st);
        case SNF_BF16: return snf::td_top_t((const __bf16*)x, R, V, ld, k, temperature, ids, (__bf16*)logits, rest, workspace, st);
        default: return snf::td_top_t((const _Float16*)x, R, V, ld, k, temperature, ids, (_Float16*)logits, rest, workspace, st);
    }
}

int64_t snf_top_distill_workspace_bytes(int R, int V, int dtype) {
    if (R < 1 || V < 1) return 0;
    const snf::TdPlan pl = snf::td_rows_plan(R, V, dtype == SNF_F32 ? 4 : 8);
    return pl.parts == 1 ? 0 : (int64_t)R * pl.parts * 8;
}

int snf_top_distill_fwd(const void* z, int dtype, int R, int V, int64_t ld, const void* ids, int ids_wide, const void* top, int top_dtype,
                        const float* rest, int K, float temperature, float weight, float* rows, float* counted, float* stats, float* diff,
                        int mean, float* loss, float* divisor, void* workspace, int64_t workspace_bytes, snf_stream_t stream) {
    SNF_REQUIRE(R >= 0 && V >= 1 && V <= SNF_TOP_MAX_V, "snf_top_distill_fwd: bad sizes R=%d V=%d", R, V);
    SNF_REQUIRE(K >= 1 && K <= snf::TD_MAX_K, "snf_top_distill_fwd: K=%d is not in 1 .. %d", K, snf::TD_MAX_K);
    SNF_REQUIRE(temperature >= FLT_MIN && temperature < INFINITY, "snf_top_distill_fwd: temperature %g", (double)temperature);
    SNF_REQUIRE(snf::td_weight_ok(weight, temperature), "snf_top_distill_fwd: weight %g (T %g): it and weight T^2 are 0 or normal numbers",
                (double)weight, (double)temperature);
    SNF_REQUIRE(dtype >= SNF_F32 && dtype <= SNF_F16 && top_dtype >= SNF_F32 && top_dtype <= SNF_F16, "snf_top_distill_fwd: unknown dtype");
    SNF_REQUIRE(!loss || divisor, "snf_top_distill_fwd: null pointer");
    hipStream_t st = (hipStream_t)stream;
    if (R == 0) return loss ? snf::td_mean(rows, counted, R, mean, loss, divisor, st) : SNF_OK;
    SNF_REQUIRE(z && ids && top && rows && counted && stats && diff, "snf_top_distill_fwd: null pointer");
    SNF_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "snf_top_distill_fwd: stats is not aligned to 8 bytes");
    SNF_REQUIRE(ld >= V || R == 1, "snf_top_distill_fwd: rows of %d values overlap at stride %lld", V, (long long)ld);
    SNF_REQUIRE(workspace_bytes >= snf_top_distill_workspace_bytes(R, V, dtype) && (workspace_bytes == 0 || workspace),
                "snf_top_distill_fwd: workspace of %lld bytes is too small", (long long)workspace_bytes);
    const snf::TdTeacher t{ids, top, rest, ids_wide, top_dtype, K};
    const snf::TdSaved out{rows, counted, (float2*)stats, diff};
#define TD_T(T_) snf::td_fwd_t<T_>((const T_*)z, R, V, ld, t, temperature, weight, out, workspace, st)
    const int rc = dtype == SNF_F32 ? TD_T(float) : dtype == SNF_BF16 ? TD_T(__bf16) : TD_T(_Float16);
#undef TD_T
    return rc != SNF_OK || !loss ? rc : snf::td_mean(rows, counted, R, mean, loss, divisor, st);
}

int snf_top_distill_bwd(const void* z, int dtype, int R, int V, int64_t ld, const void* ids, int ids_wide, int K, float temperature,
                        float weight, const float* g, int g_per_row, const float* divisor, const float* counted, const float* stats,
                        const float* diff, void* dz, snf_stream_t stream) {
    SNF_REQUIRE(R >= 0 && V >= 1 && V <= SNF_TOP_MAX_V, "snf_top_distill_bwd: bad sizes R=%d V=%d", R, V);
    SNF_REQUIRE(K >= 1 && K <= snf::TD_MAX_K, "snf_top_distill_bwd: K=%d is not in 1 .. %d", K, snf::TD_MAX_K);
    SNF_REQUIRE(temperature >= FLT_MIN && temperature < INFINITY, "snf_top_distill_bwd: temperature %g", (double)temperature);
    SNF_REQUIRE(snf::td_weight_ok(weight, temperature), "snf_top_distill_bwd: weight %g (T %g): it and weight T^2 are 0 or normal numbers",
                (double)weight, (double)temperature);
    SNF_REQUIRE(dtype >= SNF_F32 && dtype <= SNF_F16, "snf_top_distill_bwd: unknown dtype %d", dtype);
    if (R == 0) return SNF_OK;
    SNF_REQUIRE(z && ids && g && counted && stats && diff && dz, "snf_top_distill_bwd: null pointer");
    SNF_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0, "snf_top_distill_bwd: stats is not aligned to 8 bytes");
    SNF_REQUIRE(ld >= V || R == 1, "snf_top_distill_bwd: rows of %d values overlap at stride %lld", V, (long long)ld);
    hipStream_t st = (hipStream_t)stream;
    const float2* s2 = (const float2*)stats;
#define TD_T(T_) snf::td_bwd_t<T_>((const T_*)z, R, V, ld, ids, ids_wide, K, temperature, weight, g, g_per_row, divisor, counted, s2, diff, \
                                   (T_*)dz, st)
    switch (dtype) {
        case SNF_F32: return TD_T(float);
        case SNF_BF16: return TD_T(__bf16);
        default: return TD_T(_Float16);
    }
#undef TD_T
}

}  // extern "C"
