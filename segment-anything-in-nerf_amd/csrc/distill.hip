// distill.hip -- a teacher's top logits and the distillation loss that reads them (gfx950).
//   snf_top_logits     : the k largest logits of a row in order, and log sum exp(x / T) over all the others
//   snf_top_distill_*  : T^2 KL(teacher || student) per row, from the teacher's top logits (and the mass of the rest, as one class of its
//                        own), with the student's gradient
// Both read a row once: a workgroup holds its part of the row in registers (16 bytes a load, all in flight at once), so that the maximum,
// the selection and the sums of exponentials see the same registers.
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
// exp((x - m) / T), c = log2(e) / T; nothing is left of x = -inf, also where the maximum is
__device__ __forceinline__ float td_term(float x, float m, float c) { return x == TD_NINF ? 0.f : td_exp2((x - m) * c); }

struct TdMaxOp { __device__ static float op(float a, float b) { return td_max(a, b); } };
struct TdSumOp { __device__ static float op(float a, float b) { return a + b; } };
struct TdCountOp { __device__ static int op(int a, int b) { return a + b; } };

// the same value in every thread of the workgroup; `s` is scratch of one word per wave, free again after the call
template <int THREADS, typename OP, typename V>
__device__ __forceinline__ V td_reduce(V v, V* s) {
#pragma unroll
    for (int d = WAVE / 2; d > 0; d >>= 1) v = OP::op(v, __shfl_xor(v, d, WAVE));
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
    static constexpr int CAPACITY = THREADS * NV * E - E;  // elements of a part at any alignment (a multiple of E)
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
        if (threadIdx.x == 0)
            for (int e = 0; e < shift; ++e) td_clear<T>(r[0], e);
        const int last = granules - 1, over = granules * E - shift - n;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * THREADS + (int)threadIdx.x == last)
                for (int e = E - over; e < E; ++e) td_clear<T>(r[j], e);
    }
    __device__ __forceinline__ int place(int j, int e) const { return (j * THREADS + (int)threadIdx.x) * E + e - shift; }
    __device__ __forceinline__ bool inside(int place) const { return (unsigned)place < (unsigned)len; }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float x[E];
            td_unpack<T>(r[j], x);
#pragma unroll
            for (int e = 0; e < E; ++e) f(x[e], j, e);
        }
    }
};

// =================================================================================================================================
// top logits
// =================================================================================================================================
// One pass: (1) every thread's largest element; the k-th largest of G >= k group maxima is a bound that at least k elements reach and few
// others do (G = 2 k groups: about 0.7 x 2 k of them for values in random order); (2) what reaches the bound goes to LDS as 64-bit keys
// (value, place: all different, so ranks do not depend on the order of arrival), a key's rank is the number of larger keys; (3) the sum
// over the rest refers to the largest logit of the rest, so that it keeps its digits however far below the top it lies.
// Rows with a NaN and rows where more than TD_CAND elements reach the bound (long runs of equal logits) take the exact way: bisection of
// the k-th key over its bits, then of the places among its equals.
constexpr int TD_CAND = 1024;

template <typename T, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void k_top_logits(const T* __restrict__ x, int V, int64_t ld, int k, int groups, float temperature,
                                                        int parts, int part_len, int32_t* __restrict__ ids, T* __restrict__ logits,
                                                        float* __restrict__ rest, uint64_t* __restrict__ part_keys,
                                                        float2* __restrict__ part_rest) {
    constexpr int CAND = THREADS == 64 ? 256 : TD_CAND;
    __shared__ uint64_t s_key[CAND];
    __shared__ float s_group[THREADS];
    __shared__ float s_red[THREADS / WAVE];
    __shared__ uint32_t s_bound;
    __shared__ int s_n, s_equal;
    __shared__ uint64_t s_kth, s_next;
    const int row = (int)(blockIdx.x / (unsigned)parts), part = (int)(blockIdx.x % (unsigned)parts);
    const int p0 = part * part_len, len = min(part_len, V - p0);
    TdPart<T, THREADS, NV> reg;
    reg.load(x + (int64_t)row * ld + p0, len);
    const int kk = min(k, len);
    const float c = TD_LOG2E / temperature;
    if (threadIdx.x == 0) { s_bound = 0; s_n = 0; s_equal = 0; s_next = 0; }

    float own = TD_NINF;
    reg.each([&](float v, int, int) { own = td_max(own, v); });
    const float top = td_reduce<THREADS, TdMaxOp>(own, s_red);
    bool slow = top != top;
    if (!slow) {
        // groups of THREADS / groups neighbouring threads (a power of two, at most a wave)
        const int gs = THREADS / groups;
        float gm = own;
        for (int d = 1; d < gs; d <<= 1) gm = td_max(gm, __shfl_xor(gm, d, WAVE));
        if ((int)threadIdx.x % gs == 0) s_group[threadIdx.x / gs] = gm;
        __syncthreads();
        if ((int)threadIdx.x < groups) {
            const float mine = s_group[threadIdx.x];
            int ge = 0;
            for (int i = 0; i < groups; ++i) ge += s_group[i] >= mine;
            if (ge >= kk) atomicMax(&s_bound, td_key(mine));
        }
        __syncthreads();
        const float bound = td_value(s_bound);
        if (own >= bound) {
            reg.each([&](float v, int j, int e) {
                if (v >= bound) {
                    const int p = reg.place(j, e);
                    if (reg.inside(p)) {
                        const int at = atomicAdd(&s_n, 1);
                        if (at < CAND) s_key[at] = (uint64_t)td_key(v) << 32 | (uint32_t)~(p0 + p);
                    }
                }
            });
        }
        __syncthreads();
        slow = s_n > CAND;
    }
    uint32_t kth_key = 0;
    int equal_left = 0;  // (slow) elements of the rest that equal the k-th
    if (slow) {
        int* s_redi = reinterpret_cast<int*>(s_red);
        auto count = [&](auto pred) {
            int n = 0;
            reg.each([&](float v, int j, int e) {
                const int p = reg.place(j, e);
                n += reg.inside(p) && pred(td_key(v), p);
            });
            return td_reduce<THREADS, TdCountOp>(n, s_redi);
        };
        uint32_t v = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t t = v | 1u << bit;
            if (count([&](uint32_t key, int) { return key >= t; }) >= kk) v = t;
        }
        const int need = kk - count([&](uint32_t key, int) { return key > v; });
        const int equal = count([&](uint32_t key, int) { return key == v; });
        int cut = len;  // the smallest with `need` equals before it
        if (need < equal) {
            int lo = 0;
            while (lo < cut) {
                const int mid = (lo + cut) >> 1;
                if (count([&](uint32_t key, int p) { return key == v && p < mid; }) >= need) cut = mid;
                else lo = mid + 1;
            }
        }
        equal_left = equal - need;
        kth_key = v;
        __syncthreads();
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        reg.each([&](float f, int j, int e) {
            const int p = reg.place(j, e);
            const uint32_t key = td_key(f);
            if (reg.inside(p) && (key > v || (key == v && p < cut))) s_key[atomicAdd(&s_n, 1)] = (uint64_t)key << 32 | (uint32_t)~(p0 + p);
        });
        __syncthreads();
    }
    const int n = s_n;  // kk <= n <= CAND
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const uint64_t mine = s_key[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s_key[j] > mine;
        if (rank < kk) {
            if (parts == 1) {
                ids[(int64_t)row * k + rank] = (int32_t)~(uint32_t)mine;
                logits[(int64_t)row * k + rank] = (T)td_value((uint32_t)(mine >> 32));
            } else {
                part_keys[((int64_t)row * parts + part) * k + rank] = mine;
            }
            if (rank == kk - 1) s_kth = mine;
        } else if (rank == kk) {
            s_next = mine;
        }
    }
    if (parts > 1)
        for (int i = kk + threadIdx.x; i < k; i += THREADS) part_keys[((int64_t)row * parts + part) * k + i] = 0;  // a short part
    __syncthreads();
    float m, sum = 0.f;
    if (!slow) {
        const float kth = td_value((uint32_t)(s_kth >> 32));
        if (n > kk) {
            for (int i = threadIdx.x; i < n; i += THREADS)  // the candidates of the rest that equal the k-th
                if ((uint32_t)(s_key[i] >> 32) == (uint32_t)(s_kth >> 32) && s_key[i] < s_kth) atomicAdd(&s_equal, 1);
            m = td_value((uint32_t)(s_next >> 32));
            __syncthreads();
            equal_left = s_equal;
        } else {
            m = TD_NINF;
            reg.each([&](float v, int, int) { if (v < kth) m = td_max(m, v); });
            m = td_reduce<THREADS, TdMaxOp>(m, s_red);
        }
        if (m > TD_NINF)
            reg.each([&](float v, int, int) { sum += v < kth ? td_exp2((v - m) * c) : 0.f; });
    } else {
        m = equal_left > 0 ? td_value(kth_key) : TD_NINF;
        if (equal_left == 0) {
            reg.each([&](float v, int, int) { if (td_key(v) < kth_key) m = td_max(m, v); });
            m = td_reduce<THREADS, TdMaxOp>(m, s_red);
        }
        if (m != TD_NINF)
            reg.each([&](float v, int, int) { sum += td_key(v) < kth_key ? td_term(v, m, c) : 0.f; });
    }
    sum = td_reduce<THREADS, TdSumOp>(sum, s_red) + (float)equal_left;
    if (threadIdx.x == 0) {
        if (m == TD_NINF) sum = 0.f;  // nothing left, or nothing but -inf
        if (parts == 1) rest[row] = m == INFINITY || m == TD_NINF ? m : m / temperature + logf(sum);
        else part_rest[(int64_t)row * parts + part] = make_float2(m, sum);
    }
}

// the parts of a row joined: a key's rank is the sum of its places in the parts' sorted lists
template <typename T>
__global__ __launch_bounds__(256) void k_top_logits_join(int k, int parts, float temperature, const uint64_t* __restrict__ part_keys,
                                                         const float2* __restrict__ part_rest, int32_t* __restrict__ ids,
                                                         T* __restrict__ logits, float* __restrict__ rest) {
    extern __shared__ uint64_t s_keys[];
    __shared__ uint64_t s_next;
    __shared__ float s_red[4];
    const int row = blockIdx.x, n = parts * k;
    const float c = TD_LOG2E / temperature;
    if (threadIdx.x == 0) s_next = 0;
    for (int i = threadIdx.x; i < n; i += 256) s_keys[i] = part_keys[(int64_t)row * n + i];
    __syncthreads();
    uint32_t lost = 0;  // bit q: this thread's q-th key belongs to the rest (n <= 32 * 256)
    for (int i = threadIdx.x, q = 0; i < n; i += 256, ++q) {
        const uint64_t mine = s_keys[i];
        if (mine == 0) continue;  // a short part's filling
        int rank = 0;
        for (int p = 0; p < parts; ++p) {
            int lo = 0, hi = k;  // keys of part p above `mine`
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s_keys[p * k + mid] > mine) lo = mid + 1; else hi = mid;
            }
            rank += lo;
        }
        if (rank < k) {
            ids[(int64_t)row * k + rank] = (int32_t)~(uint32_t)mine;
            logits[(int64_t)row * k + rank] = (T)td_value((uint32_t)(mine >> 32));
        } else {
            lost |= 1u << q;
            if (rank == k) s_next = mine;
        }
    }
    __syncthreads();
    float m = s_next ? td_value((uint32_t)(s_next >> 32)) : TD_NINF;
    for (int p = threadIdx.x; p < parts; p += 256) m = td_max(m, part_rest[(int64_t)row * parts + p].x);
    m = td_reduce<256, TdMaxOp>(m, s_red);
    float sum = 0.f;
    if (m != TD_NINF) {
        for (int i = threadIdx.x, q = 0; i < n; i += 256, ++q)
            if (lost >> q & 1u) sum += td_term(td_value((uint32_t)(s_keys[i] >> 32)), m, c);
        for (int p = threadIdx.x; p < parts; p += 256) {
            const float2 pr = part_rest[(int64_t)row * parts + p];
            sum += pr.y * td_term(pr.x, m, c);
        }
    }
    sum = td_reduce<256, TdSumOp>(sum, s_red);
    if (threadIdx.x == 0) rest[row] = m == INFINITY || m == TD_NINF ? m : m / temperature + logf(sum);
}

// =================================================================================================================================
// distillation loss
// =================================================================================================================================
// z [V] a student's logits, ids / t [K] the teacher's top logits (a negative id: no entry), optionally r = log sum exp(t_v / T) over all
// other places.  p = softmax over (t / T [, r]), q = softmax(z / T), q_rest = the sum of q over the places that ids does not name:
//     loss = T^2 [ sum_k p_k (log p_k - log q_{id_k}) + p_rest (log p_rest - log q_rest) ]
//     dloss / dz_v = T [ q_v - sum_{k: id_k = v} p_k - (v not named) p_rest q_v / q_rest ]
// With r the sum over the places that are not named is taken by itself, relative to its own maximum: nothing is ever subtracted from 1.
// What the backward pass needs of a row (32 + 4 K bytes): its reference m_r, the factor f with dz_v = gs f exp((z_v - m_r) / T) for all
// places that are not named, the row's maximum m, 1 / sum exp((z - m) / T), and p.
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
    float4* stats;   // [R] m_r, f, m, 1 / sum
    float* p;        // [R, K]
};

// One wave: the row's teacher side and its loss, from the student's maximum and sum (over the places that are not named where REST).
template <typename T, bool REST>
__device__ __forceinline__ void td_finish_row(const T* __restrict__ zrow, int V, int64_t row, const TdTeacher& t, float temperature,
                                              float scale, float m_r, float s_r, const TdSaved& out) {
    constexpr int Q = TD_MAX_K / WAVE;
    const int lane = lane_id();
    const float c = TD_LOG2E / temperature;
    int64_t id[Q];
    float tv[Q], zv[Q];
    bool bad = false, any = false;
    float tm = TD_NINF;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int k = q * WAVE + lane;
        id[q] = -1;
        tv[q] = zv[q] = TD_NINF;
        if (k < t.K) {
            const int64_t i = td_id(t.ids, t.ids_wide, row * t.K + k);
            bad |= i >= V;
            if (i >= 0 && i < V) {
                id[q] = i;
                any = true;
                zv[q] = (float)zrow[i];
                const float l = td_load(t.logits, t.dtype, row * t.K + k);
                tv[q] = REST ? l / temperature : l;
                tm = td_max(tm, tv[q]);
            }
        }
    }
    bad = __any(bad);
    any = __any(any) || bad;
#pragma unroll
    for (int d = WAVE / 2; d > 0; d >>= 1) tm = td_max(tm, __shfl_xor(tm, d, WAVE));
    const float r = REST ? t.rest[row] : TD_NINF;
    if (REST) tm = td_max(tm, r);
    if (!any || (tm == TD_NINF && !bad)) {  // no target: no entry, or a teacher without any mass
        if (lane == 0) {
            out.rows[row] = 0.f;
            out.counted[row] = 0.f;
            out.stats[row] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int k = lane; k < t.K; k += WAVE) out.p[row * t.K + k] = 0.f;
        return;
    }
    // teacher
    float pe[Q], ps = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        tv[q] = REST ? tv[q] - tm : (tv[q] - tm) / temperature;
        pe[q] = id[q] >= 0 ? expf(tv[q]) : 0.f;
        ps += pe[q];
    }
    ps = wave_sum(ps);
    const float re = REST ? expf(r - tm) : 0.f;
    ps += re;
    const float log_ps = logf(ps);
    // student
    float m = m_r, s = s_r;
    if (REST) {  // the named places, each once
        float nm = TD_NINF;
#pragma unroll
        for (int q = 0; q < Q; ++q) nm = td_max(nm, zv[q]);
#pragma unroll
        for (int d = WAVE / 2; d > 0; d >>= 1) nm = td_max(nm, __shfl_xor(nm, d, WAVE));
        m = td_max(m_r, nm);
        float sn = 0.f;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            if (q * WAVE >= t.K) break;
            bool first = id[q] >= 0;
#pragma unroll
            for (int q2 = 0; q2 <= q; ++q2)
                for (int l = 0; l < (q2 < q ? WAVE : WAVE - 1); ++l) {
                    if (q2 * WAVE + l >= t.K) break;
                    const int other = __shfl((int)id[q2], l, WAVE);
                    if (q2 * WAVE + l < q * WAVE + lane && other == (int)id[q]) first = false;
                }
            if (first) sn += td_term(zv[q], m, c);
        }
        s = wave_sum(sn) + s_r * td_term(m_r, m, c);
    }
    const float log_s = logf(s);
    float loss = 0.f;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int k = q * WAVE + lane;
        const float p = pe[q] / ps;
        if (k < t.K) out.p[row * t.K + k] = p;
        if (id[q] >= 0 && (p > 0.f || p != p)) loss += p * ((tv[q] - log_ps) - ((zv[q] - m) / temperature - log_s));
    }
    loss = wave_sum(loss);
    float f = 1.f / s, ref = m;
    if (REST) {
        const float pr = re / ps;
        if (pr > 0.f || pr != pr) loss += pr * ((r - tm - log_ps) - ((m_r - m) / temperature + logf(s_r) - log_s));
        ref = m_r;
        f = td_term(m_r, m, c) / s - (pr > 0.f || pr != pr ? pr / s_r : 0.f);
        if (m_r == TD_NINF) { ref = 0.f; f = 0.f; }  // every place is named, or what is not is -inf
    }
    if (bad) loss = f = __uint_as_float(0x7FC00000u);  // an id past the end
    if (lane == 0) {
        out.rows[row] = loss * scale;
        out.counted[row] = 1.f;
        out.stats[row] = make_float4(ref, f, m, bad ? f : 1.f / s);
    }
}

template <typename T, bool REST, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void k_top_distill_rows(const T* __restrict__ z, int V, int64_t ld, TdTeacher t, float temperature,
                                                              float scale, int parts, int part_len, TdSaved out,
                                                              float2* __restrict__ part_ms) {
    using Part = TdPart<T, THREADS, NV>;
    constexpr int WORDS = (THREADS * NV * Part::E + 31) / 32;
    __shared__ uint32_t s_named[REST ? WORDS : 1];
    __shared__ float s_red[THREADS / WAVE];
    const int64_t row = blockIdx.x / (unsigned)parts;
    const int part = (int)(blockIdx.x % (unsigned)parts);
    const int p0 = part * part_len, len = min(part_len, V - p0);
    const T* zrow = z + row * ld;
    Part reg;
    reg.load(zrow + p0, len);
    if (REST) {  // the named places become -inf: one bit per place of the part, in the order of the registers
        for (int i = threadIdx.x; i < WORDS; i += THREADS) s_named[i] = 0;
        __syncthreads();
        for (int k = threadIdx.x; k < t.K; k += THREADS) {
            const int64_t i = td_id(t.ids, t.ids_wide, row * t.K + k) - p0;
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
        td_finish_row<T, REST>(zrow, V, row, t, temperature, scale, m, s, out);
    }
}

// rows in parts: the parts' maxima and sums joined, then the row as above; one wave per row
template <typename T, bool REST>
__global__ __launch_bounds__(64) void k_top_distill_join(const T* __restrict__ z, int V, int64_t ld, TdTeacher t, float temperature,
                                                         float scale, int parts, TdSaved out, const float2* __restrict__ part_ms) {
    const int64_t row = blockIdx.x;
    const float c = TD_LOG2E / temperature;
    float m = TD_NINF, s = 0.f;
    for (int p = lane_id(); p < parts; p += WAVE) m = td_max(m, part_ms[row * parts + p].x);
#pragma unroll
    for (int d = WAVE / 2; d > 0; d >>= 1) m = td_max(m, __shfl_xor(m, d, WAVE));
    for (int p = lane_id(); p < parts; p += WAVE) {
        const float2 ms = part_ms[row * parts + p];
        s += ms.y * td_term(ms.x, m, c);
    }
    s = wave_sum(s);
    td_finish_row<T, REST>(z + row * ld, V, row, t, temperature, scale, m, s, out);
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
                                                         const float* __restrict__ counted, const float4* __restrict__ stats,
                                                         const float* __restrict__ p, T* __restrict__ dz) {
    constexpr int E = 16 / (int)sizeof(T);
    __shared__ uint32_t s_named[TD_CHUNK / 32 + 1];
    __shared__ int s_id[TD_MAX_K];
    __shared__ float s_p[TD_MAX_K];
    const int64_t row = blockIdx.x / (unsigned)chunks;
    const int p0 = (int)(blockIdx.x % (unsigned)chunks) * TD_CHUNK, len = min(TD_CHUNK, V - p0);
    const T* zp = z + row * ld + p0;
    T* dp = dz + row * V + p0;
    const bool live = counted[row] != 0.f;
    const float gs = g[g_per_row ? row : 0] * scale / (divisor ? divisor[0] : 1.f);
    const float c = TD_LOG2E / temperature;
    const float4 st = stats[row];
    const float f = gs * st.y;
    if (live) {
        for (int i = threadIdx.x; i < TD_CHUNK / 32 + 1; i += blockDim.x) s_named[i] = 0;
        __syncthreads();
    }
    const int shift = PACKED ? (int)((reinterpret_cast<uintptr_t>(zp) & 15) / sizeof(T)) : 0;
    if (live) {
        for (int k = threadIdx.x; k < K; k += blockDim.x) {
            const int64_t i = td_id(ids, ids_wide, row * K + k) - p0;
            const bool here = i >= 0 && i < len;
            s_id[k] = here ? (int)i : -1;
            s_p[k] = p[row * K + k];
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
                    sum += s_p[o];
                }
            if (first) dp[i] = (T)(gs * (td_exp2(((float)zp[i] - st.z) * c) * st.w - sum));
        }
    }
    if constexpr (PACKED) {
        const uint4* zg = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(zp) & ~(uintptr_t)15);
        uint4* dg = reinterpret_cast<uint4*>(reinterpret_cast<uintptr_t>(dp) & ~(uintptr_t)15);
        const int granules = (shift + len + E - 1) / E;
        for (int v = threadIdx.x; v < granules; v += blockDim.x) {
            float x[E];
            struct alignas(16) { T v[E]; } o;
            if (live) {
                td_unpack<T>(zg[v], x);
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = (T)(f * td_exp2((x[e] - st.x) * c));
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = (T)0.f;
            }
            const int b = v * E;
            const uint32_t bits = live ? s_named[b >> 5] >> (b & 31) & ((1u << E) - 1u) : 0u;
            if (bits == 0 && b >= shift && b + E <= shift + len) {
                dg[v] = *reinterpret_cast<const uint4*>(&o);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (!(bits >> e & 1u) && b + e >= shift && b + e < shift + len) dp[b + e - shift] = o.v[e];
            }
        }
    } else {
        for (int i = threadIdx.x; i < len; i += blockDim.x)
            if (!live) dp[i] = (T)0.f;
            else if (!(s_named[i >> 5] >> (i & 31) & 1u)) dp[i] = (T)(f * td_exp2(((float)zp[i] - st.x) * c));
    }
}

// ---- launch shapes ----------------------------------------------------------------------------------------------------------------
// shapes a row (or a part of it) is held in, smallest first: threads x 16-byte granules a thread
struct TdShape { int threads, nv; };
constexpr TdShape TD_SHAPES[] = {{64, 1}, {64, 4}, {256, 4}, {256, 16}, {512, 16}};
constexpr int TD_NSHAPES = 5;

struct TdPlan { int shape, parts, part_len; };

// The smallest shape that holds a row; where that leaves most of the chip idle (fewer than 256 workgroups), smaller parts of a row per
// workgroup and a join -- down to the wave of four granules, and to no more parts than `max_parts`.
static TdPlan td_plan(int R, int V, int E, int min_threads, int max_parts) {
    auto cap = [&](int s) { return TD_SHAPES[s].threads * TD_SHAPES[s].nv * E - E; };
    int s = 0;
    while (s + 1 < TD_NSHAPES && (cap(s) < V || TD_SHAPES[s].threads < min_threads)) ++s;
    int parts = ceil_div(V, cap(s));
    while (s > 1 && TD_SHAPES[s - 1].threads >= min_threads && (long long)R * parts < 256 && ceil_div(V, cap(s - 1)) <= max_parts) {
        --s;
        parts = ceil_div(V, cap(s));
    }
    return {s, parts, parts == 1 ? V : cap(s)};
}

static TdPlan td_top_plan(int R, int V, int k, int E) {
    // 2 k threads where there are as many (the bound is the k-th of the groups' maxima); at most 1024 keys to join unless the row is
    // longer than 1024 / k parts of the largest shape (V <= SNF_TOP_MAX_V: at most 32 parts, 8192 keys, 64 KB)
    return td_plan(R, V, E, k <= 32 ? 64 : k <= 128 ? 256 : 512, 1024 / k);
}

template <typename T>
static int td_top_t(const T* x, int R, int V, int64_t ld, int k, float temperature, int32_t* ids, T* logits, float* rest, void* ws,
                    hipStream_t st) {
    const TdPlan pl = td_top_plan(R, V, k, 16 / (int)sizeof(T));
    SNF_REQUIRE((int64_t)R * pl.parts * TD_SHAPES[pl.shape].threads < ((int64_t)1 << 32), "snf_top_logits: %d rows of %d are too many for one launch", R, V);
    uint64_t* keys = (uint64_t*)ws;
    float2* pr = (float2*)(keys + (size_t)R * pl.parts * k);
    const int threads = TD_SHAPES[pl.shape].threads;
    int groups = 32;
    while (groups < 2 * k) groups *= 2;
    if (groups > threads) groups = threads;
    if (threads / groups > WAVE) groups = threads / WAVE;
    const dim3 grid((unsigned)((int64_t)R * pl.parts));
#define TD_GO(S_)                                                                                                                     \
    case S_:                                                                                                                          \
        k_top_logits<T, TD_SHAPES[S_].threads, TD_SHAPES[S_].nv><<<grid, dim3(TD_SHAPES[S_].threads), 0, st>>>(                       \
            x, V, ld, k, groups, temperature, pl.parts, pl.part_len, ids, logits, rest, keys, pr);                                    \
        break;
    switch (pl.shape) { TD_GO(0) TD_GO(1) TD_GO(2) TD_GO(3) TD_GO(4) }
#undef TD_GO
    SNF_LAUNCH_CHECK("snf_top_logits");
    if (pl.parts > 1) {
        k_top_logits_join<T><<<dim3(R), dim3(256), (size_t)pl.parts * k * 8, st>>>(k, pl.parts, temperature, keys, pr, ids, logits, rest);
        SNF_LAUNCH_CHECK("snf_top_logits (join)");
    }
    return SNF_OK;
}

template <typename T, bool REST>
static int td_fwd_t(const T* z, int R, int V, int64_t ld, const TdTeacher& t, float temperature, float weight, const TdSaved& out, void* ws,
                    hipStream_t st) {
    const TdPlan pl = td_plan(R, V, 16 / (int)sizeof(T), 64, 1 << 30);
    SNF_REQUIRE((int64_t)R * pl.parts * TD_SHAPES[pl.shape].threads < ((int64_t)1 << 32), "snf_top_distill_fwd: %d rows of %d are too many for one launch", R, V);
    const float scale = weight * temperature * temperature;
    const dim3 grid((unsigned)((int64_t)R * pl.parts));
#define TD_GO(S_)                                                                                                                     \
    case S_:                                                                                                                          \
        k_top_distill_rows<T, REST, TD_SHAPES[S_].threads, TD_SHAPES[S_].nv><<<grid, dim3(TD_SHAPES[S_].threads), 0, st>>>(           \
            z, V, ld, t, temperature, scale, pl.parts, pl.part_len, out, (float2*)ws);                                                \
        break;
    switch (pl.shape) { TD_GO(0) TD_GO(1) TD_GO(2) TD_GO(3) TD_GO(4) }
#undef TD_GO
    SNF_LAUNCH_CHECK("snf_top_distill_fwd");
    if (pl.parts > 1) {
        k_top_distill_join<T, REST><<<dim3(R), dim3(64), 0, st>>>(z, V, ld, t, temperature, scale, pl.parts, out, (const float2*)ws);
        SNF_LAUNCH_CHECK("snf_top_distill_fwd (join)");
    }
    return SNF_OK;
}

template <typename T>
static int td_bwd_t(const T* z, int R, int V, int64_t ld, const void* ids, int ids_wide, int K, float temperature, float weight,
                    const float* g, int g_per_row, const float* divisor, const float* counted, const float4* stats, const float* p, T* dz,
                    hipStream_t st) {
    const int chunks = ceil_div(V, TD_CHUNK);
    SNF_REQUIRE((int64_t)R * chunks * 256 < ((int64_t)1 << 32), "snf_top_distill_bwd: %d rows of %d are too many for one launch", R, V);
    const dim3 grid((unsigned)((int64_t)R * chunks)), block(V <= 1024 ? 64 : 256);
    const size_t zb = ((size_t)ld * sizeof(T)) % 16, db = ((size_t)V * sizeof(T)) % 16;
    const bool packed = (R == 1 || zb == db) && (reinterpret_cast<uintptr_t>(z) & 15) == (reinterpret_cast<uintptr_t>(dz) & 15);
    if (packed)
        k_top_distill_bwd<T, true><<<grid, block, 0, st>>>(z, V, ld, ids, ids_wide, K, temperature, weight * temperature, chunks, g, g_per_row,
                                                           divisor, counted, stats, p, dz);
    else
        k_top_distill_bwd<T, false><<<grid, block, 0, st>>>(z, V, ld, ids, ids_wide, K, temperature, weight * temperature, chunks, g,
                                                            g_per_row, divisor, counted, stats, p, dz);
    SNF_LAUNCH_CHECK("snf_top_distill_bwd");
    return SNF_OK;
}

}  // namespace snf

extern "C" {

int64_t snf_top_logits_workspace_bytes(int R, int V, int k, int dtype) {
    if (R < 1 || V < 1 || k < 1 || k > snf::TD_MAX_K || k > V) return 0;
    const snf::TdPlan pl = snf::td_top_plan(R, V, k, dtype == SNF_F32 ? 4 : 8);
    return pl.parts == 1 ? 0 : (int64_t)R * pl.parts * (8 * (int64_t)k + 8);
}

int snf_top_logits(const void* x, int dtype, int R, int V, int64_t ld, int k, float temperature, int32_t* ids, void* logits, float* rest,
                   void* workspace, int64_t workspace_bytes, snf_stream_t stream) {
    SNF_REQUIRE(R >= 0 && V >= 1 && V <= SNF_TOP_MAX_V, "snf_top_logits: bad sizes R=%d V=%d", R, V);
    SNF_REQUIRE(k >= 1 && k <= snf::TD_MAX_K && k <= V, "snf_top_logits: k=%d is not in 1 .. min(V, %d)", k, snf::TD_MAX_K);
    SNF_REQUIRE(temperature > 0.f && temperature < INFINITY, "snf_top_logits: temperature %g", (double)temperature);
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
    const snf::TdPlan pl = snf::td_plan(R, V, dtype == SNF_F32 ? 4 : 8, 64, 1 << 30);
    return pl.parts == 1 ? 0 : (int64_t)R * pl.parts * 8;
}

int snf_top_distill_fwd(const void* z, int dtype, int R, int V, int64_t ld, const void* ids, int ids_wide, const void* top, int top_dtype,
                        const float* rest, int K, float temperature, float weight, float* rows, float* counted, float* stats, float* p,
                        void* workspace, int64_t workspace_bytes, snf_stream_t stream) {
    SNF_REQUIRE(R >= 0 && V >= 1 && V <= SNF_TOP_MAX_V, "snf_top_distill_fwd: bad sizes R=%d V=%d", R, V);
    SNF_REQUIRE(K >= 1 && K <= snf::TD_MAX_K, "snf_top_distill_fwd: K=%d is not in 1 .. %d", K, snf::TD_MAX_K);
    SNF_REQUIRE(temperature > 0.f && temperature < INFINITY, "snf_top_distill_fwd: temperature %g", (double)temperature);
    SNF_REQUIRE(dtype >= SNF_F32 && dtype <= SNF_F16 && top_dtype >= SNF_F32 && top_dtype <= SNF_F16, "snf_top_distill_fwd: unknown dtype");
    if (R == 0) return SNF_OK;
    SNF_REQUIRE(z && ids && top && rows && counted && stats && p, "snf_top_distill_fwd: null pointer");
    SNF_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, "snf_top_distill_fwd: stats is not aligned to 16 bytes");
    SNF_REQUIRE(ld >= V || R == 1, "snf_top_distill_fwd: rows of %d values overlap at stride %lld", V, (long long)ld);
    SNF_REQUIRE(workspace_bytes >= snf_top_distill_workspace_bytes(R, V, dtype) && (workspace_bytes == 0 || workspace),
                "snf_top_distill_fwd: workspace of %lld bytes is too small", (long long)workspace_bytes);
    hipStream_t st = (hipStream_t)stream;
    const snf::TdTeacher t{ids, top, rest, ids_wide, top_dtype, K};
    const snf::TdSaved out{rows, counted, (float4*)stats, p};
#define TD_T(T_) (rest ? snf::td_fwd_t<T_, true>((const T_*)z, R, V, ld, t, temperature, weight, out, workspace, st)                  \
                       : snf::td_fwd_t<T_, false>((const T_*)z, R, V, ld, t, temperature, weight, out, workspace, st))
    switch (dtype) {
        case SNF_F32: return TD_T(float);
        case SNF_BF16: return TD_T(__bf16);
        default: return TD_T(_Float16);
    }
#undef TD_T
}

int snf_top_distill_mean(const float* rows, const float* counted, int R, int mean, float* loss, float* divisor,
                         snf_stream_t stream) {
    SNF_REQUIRE(R >= 0, "snf_top_distill_mean: bad size R=%d", R);
    SNF_REQUIRE(loss && divisor && (R == 0 || (rows && counted)), "snf_top_distill_mean: null pointer");
    snf::k_top_distill_mean<<<dim3(1), dim3(1024), 0, (hipStream_t)stream>>>(rows, counted, R, mean, loss, divisor);
    SNF_LAUNCH_CHECK("snf_top_distill_mean");
    return SNF_OK;
}

int snf_top_distill_bwd(const void* z, int dtype, int R, int V, int64_t ld, const void* ids, int ids_wide, int K, float temperature,
                        float weight, const float* g, int g_per_row, const float* divisor, const float* counted, const float* stats,
                        const float* p, void* dz, snf_stream_t stream) {
    SNF_REQUIRE(R >= 0 && V >= 1 && V <= SNF_TOP_MAX_V, "snf_top_distill_bwd: bad sizes R=%d V=%d", R, V);
    SNF_REQUIRE(K >= 1 && K <= snf::TD_MAX_K, "snf_top_distill_bwd: K=%d is not in 1 .. %d", K, snf::TD_MAX_K);
    SNF_REQUIRE(temperature > 0.f && temperature < INFINITY, "snf_top_distill_bwd: temperature %g", (double)temperature);
    SNF_REQUIRE(dtype >= SNF_F32 && dtype <= SNF_F16, "snf_top_distill_bwd: unknown dtype %d", dtype);
    if (R == 0) return SNF_OK;
    SNF_REQUIRE(z && ids && g && counted && stats && p && dz, "snf_top_distill_bwd: null pointer");
    SNF_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 15) == 0, "snf_top_distill_bwd: stats is not aligned to 16 bytes");
    SNF_REQUIRE(ld >= V || R == 1, "snf_top_distill_bwd: rows of %d values overlap at stride %lld", V, (long long)ld);
    hipStream_t st = (hipStream_t)stream;
    const float4* s4 = (const float4*)stats;
#define TD_T(T_) snf::td_bwd_t<T_>((const T_*)z, R, V, ld, ids, ids_wide, K, temperature, weight, g, g_per_row, divisor, counted, s4, p,   \
                                   (T_*)dz, st)
    switch (dtype) {
        case SNF_F32: return TD_T(float);
        case SNF_BF16: return TD_T(__bf16);
        default: return TD_T(_Float16);
    }
#undef TD_T
}

}  // extern "C"
