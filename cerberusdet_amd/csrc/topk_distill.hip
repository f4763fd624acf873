// Distillation from a teacher's top k logits on logits that are in memory: loss and gradient of every row in one launch.
//   p = softmax(z / tau) over the row's V logits, q = softmax of the teacher's filled slots / tau
//   loss = tau^2 sum_j q_j (log q_j - log p[idx_j]),   dz_v = drow * grad_scale * tau * (p_v - sum_{j: idx_j == v} q_j)
// Bound by memory: logits once in, gradient once out. A row of up to 32768 logits stays in the registers of its 1, 2, 4, 8 or 16 waves, so the
// maximum, the sum and the gradient are taken from one read (td_wave_kernel, td_wide_kernel); one of up to 256 KiB is held as it is stored
// (td_held_kernel); a longer one is read again for its gradient (td_long_kernel). Above 2048 logits the gradient is written dense and then, behind a
// barrier, the k named entries are written again with their q; shorter rows put q together in LDS first. Rows of at most 128 logits (box distributions,
// ordinary class lists) take 4, 8 or 16 lanes each (td_narrow_kernel). p is exp2((z - max) c) / sum: its error does not
// grow with |z|.
#include "common.h"

namespace cdet {

constexpr float kTdLog2e = 1.4426950408889634f, kTdLn2 = 0.6931471805599453f;

struct TdArgs {
    const void* z;
    void* dz;  // null: loss only
    const int32_t* idx;
    const void* val;
    const float* drow;
    float* loss;
    uint8_t* part;  // null, or 1 where the row takes part
    int64_t ld, gld;
    int64_t rows, row0;  // row0: the launch's first
    int G, V, k, vdt;
    float c, itau, tau2, gs;  // log2(e) / tau, 1 / tau, tau^2, grad_scale * tau
};

template <int DT> struct TdElem;
template <> struct TdElem<CDET_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
template <> struct TdElem<CDET_BF16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(T v) { return bf16_bits_to_f32(v); }
    static __device__ __forceinline__ T put(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <> struct TdElem<CDET_F16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(T v) { return f16_bits_to_f32(v); }
    static __device__ __forceinline__ T put(float v) { return f32_to_f16_bits(v); }
};
// N elements at any element-aligned address (the memory path takes unaligned vectors)
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) TdVec {
    T v[N];
};

// exponential of a logit relative to the row's maximum, the one form that sums, loss and gradient share: the difference first, so that the error does not grow
// with |z| (one fused rounding of z c, for 16-bit logits, put the sum and the named entries 13 nats apart at -1e9, and z c leaves fp32's range before z does;
// no slower but in td_held_kernel, which has its own)
__device__ __forceinline__ float td_exp2(float z, float mu, float c) { return __builtin_amdgcn_exp2f((z - mu) * c); }
typedef __attribute__((ext_vector_type(2))) float tdf2;
typedef __attribute__((ext_vector_type(2))) __bf16 tdb2;
typedef __attribute__((ext_vector_type(2))) _Float16 tdh2;
template <int GDT, int N>
__device__ __forceinline__ void td_put(typename TdElem<GDT>::T* dst, const float (&v)[N]) {  // N consecutive elements, converted in pairs
    if (GDT == CDET_F32) {
        TdVec<float, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = v[e];
        *reinterpret_cast<TdVec<float, N>*>(dst) = o;
    } else {
        TdVec<uint16_t, N> o;
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const uint32_t p = GDT == CDET_BF16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(tdf2{v[e], v[e + 1]}, tdb2))
                                                : __builtin_bit_cast(uint32_t, __builtin_convertvector(tdf2{v[e], v[e + 1]}, tdh2));
            __builtin_memcpy(&o.v[e], &p, 4);
        }
        *reinterpret_cast<TdVec<uint16_t, N>*>(dst) = o;
    }
}

// maximum / sum over 4, 8 or 16 neighbouring lanes: the same value in each of them
template <int L, bool MAX>
__device__ __forceinline__ float td_lanes(float v) {
#define CDET_DPP(ctrl)                                                                                                                              \
    do {                                                                                                                                            \
        const float u = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, true)); \
        v = MAX ? fmaxf(v, u) : v + u;                                                                                                              \
    } while (0)
    CDET_DPP(0xB1);   // quad_perm [1,0,3,2]
    CDET_DPP(0x4E);   // quad_perm [2,3,0,1]
    if (L > 4) CDET_DPP(0x141);  // row_half_mirror
    if (L > 8) CDET_DPP(0x140);  // row_mirror
#undef CDET_DPP
    return v;
}
// maxima / sums over a row's waves (NW = 1: inside the wave), the same value in every thread, in a fixed order
template <int NW, bool MAX>
__device__ __forceinline__ float td_reduce(float v, float* scratch) {
    v = td_lanes<16, MAX>(v);
    float u[4];  // (v_readlane: no LDS crossbar)
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 16 * i));
    v = MAX ? fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])) : (u[0] + u[1]) + (u[2] + u[3]);
    if (NW > 1) {
        const int w = (int)threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) scratch[w] = v;
        __syncthreads();
        v = scratch[0];
#pragma unroll
        for (int i = 1; i < NW; ++i) v = MAX ? fmaxf(v, scratch[i]) : v + scratch[i];
    }
    return v;
}
template <int NW>
__device__ __forceinline__ void td_sync() {
    if (NW > 1) __syncthreads();
    else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    }
}

__device__ __forceinline__ void td_row_out(const TdArgs& a, int64_t row, bool on, float sum) {
    a.loss[row] = on ? sum * a.tau2 : 0.f;
    if (a.part) a.part[row] = on;
}
// what exponents are taken relative to: the maximum, or 0 where there is nothing but -inf and NaN -- a sum of 0 then says that nothing is left, NaN stays NaN
__device__ __forceinline__ float td_base(float m) { return m == -INFINITY ? 0.f : m; }

// a row's teacher in LDS: class (-1: an empty slot), q, log q, and the student's logit there (taken before the gradient may overwrite it)
struct TdSlots {
    float *q, *lq, *z;
    int* v;
    static __host__ __device__ constexpr int up(int k) { return (k + 3) & ~3; }  // (empty ones up to the next four)
    __device__ TdSlots(float* lds, int k) : q(lds), lq(lds + up(k)), z(lds + 2 * up(k)), v(reinterpret_cast<int*>(lds + 3 * up(k))) {}
};
// fills it; t = thread of the row. False: no filled slot, or nothing but -inf in them (the sum is 0; NaN makes it NaN, which the maximum would not show)
template <int DT, int NW>
__device__ __forceinline__ bool td_teacher(const TdArgs& a, int64_t row, int t, const typename TdElem<DT>::T* z, TdSlots s, float* scratch) {
    constexpr int NT = NW * 64;
    float m = -INFINITY;
    if (t < TdSlots::up(a.k) - a.k) s.v[a.k + t] = -1;
    for (int j = t; j < a.k; j += NT) {
        int v = a.idx[row * a.k + j];
        const float x = load_elem(a.val, row * a.k + j, a.vdt) * a.itau;
        if ((unsigned)v >= (unsigned)a.V) v = -1;
        s.v[j] = v;
        s.lq[j] = x;
        if (v >= 0) {
            s.z[j] = TdElem<DT>::get(z[v]);
            m = fmaxf(m, x);
        }
    }
    m = td_base(td_reduce<NW, true>(m, scratch));
    float sum = 0.f;
    for (int j = t; j < a.k; j += NT)
        if (s.v[j] >= 0) sum += expf(s.lq[j] - m);
    sum = td_reduce<NW, false>(sum, scratch);
    const float ls = logf(sum);
    for (int j = t; j < a.k; j += NT) {
        const float lq = s.lq[j] - m - ls;
        s.lq[j] = lq;
        s.q[j] = s.v[j] >= 0 ? expf(lq) : 0.f;
    }
    return sum != 0.f;
}

// the row's loss, and the named entries of its gradient (a class named twice takes both q; the slot that names it first writes)
template <int GDT, int NW>
__device__ __forceinline__ void td_finish(const TdArgs& a, int64_t row, int t, bool on, typename TdElem<GDT>::T* dz, float mu, float inv, float l2s, float g,
                                          TdSlots s, float* scratch) {
    constexpr int NT = NW * 64;
    float sum = 0.f;
    for (int j = t; j < a.k; j += NT) {
        const int v = s.v[j];
        if (!on || v < 0) continue;
        float q = s.q[j];
        const float below = s.z[j] - mu;
        if (q != 0.f) sum += q * (s.lq[j] - (below * a.itau - l2s * kTdLn2));  // (not by way of log2 units, which end before fp32 does)
        if (!dz) continue;
        bool first = true;
        for (int o = 0; o < a.k; o += 4) {
            const int4 c = *reinterpret_cast<const int4*>(s.v + o);
            const int named[4] = {c.x, c.y, c.z, c.w};
            bool hit = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) hit = hit || (named[e] == v && o + e != j);
            if (hit)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool same = named[e] == v;
                    first = first && !(same && o + e < j);
                    q += same && o + e > j ? s.q[o + e] : 0.f;
                }
        }
        if (first) dz[v] = TdElem<GDT>::put((__builtin_amdgcn_exp2f(below * a.c) * inv - q) * g);
    }
    sum = td_reduce<NW, false>(sum, scratch);
    if (t == 0) td_row_out(a, row, on, sum);
}

template <typename T, typename TG>
__device__ __forceinline__ void td_row(const TdArgs& a, int64_t row, const T*& z, TG*& dz) {
    const unsigned px = a.G == 1 ? (unsigned)row : (unsigned)row / (unsigned)a.G, gr = (unsigned)row - px * (unsigned)a.G;  // (rows < 2^31)
    z = (const T*)a.z + (int64_t)px * a.ld + (int64_t)gr * a.V;
    dz = a.dz ? (TG*)a.dz + (int64_t)px * a.gld + (int64_t)gr * a.V : nullptr;
}

// V <= 2048: a wave a row, four rows a workgroup, the logits in registers (up to PER a lane) and, as they are stored, in LDS: the slots find theirs there, and
// then leave their numbers (16 bits) there for the dense gradient to take their q along -- no gather from and no second write to memory (67200 x 1203 fp32,
// k = 32 scattered classes: 122 us = 5.4 TB/s, with them 170). LDS of 32 bits an element leaves 16-bit rows half of the waves (67200 x 2048 bf16: 101 us =
// 5.4 TB/s, so 144). What a row holds behind its last whole 16 bytes goes a logit a lane (67200 x 1203: as a partial chunk 134 us). PER = 32 for all
// lengths: 67200 x 365 bf16 54 us, with 8 51; x 700 65, with 16 63. Addresses off by 2 bytes cost little: 67200 x 1203 bf16 75 us, x 1204 74.
__host__ __device__ constexpr int td_wave_slots(int k) { return (14 * k + 4 + 15) & ~15; }  // bytes of a row: q (k + 1), log q, the student's logits, classes,
template <typename T>
__host__ __device__ constexpr int td_wave_lds(int k, int V) {  // and the logits as they are stored (16 KiB at most)
    return td_wave_slots(k) + ((V * (int)sizeof(T) + 15) & ~15);
}
template <int DT, int GDT, int PER>
__global__ __launch_bounds__(256) void td_wave_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int CH = 16 / sizeof(T), NCH = PER / CH;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const int t = (int)threadIdx.x & 63, V = a.V, k = a.k;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
    if (row >= a.rows) return;  // (whole waves, and no barrier of the workgroup follows)
    float* const base = lds + ((int)threadIdx.x >> 6) * (td_wave_lds<T>(k, V) / 4);
    float *const sq = base, *const slq = base + k + 1, *const sz = slq + k;  // (sq[k] = 0: what a class takes that no slot names)
    int16_t* const sv = reinterpret_cast<int16_t*>(sz + k);
    T* const rb = reinterpret_cast<T*>(base + td_wave_slots(k) / 4);
    const T* z;
    TG* dz;
    td_row(a, row, z, dz);

    int v0 = -1;
    float x0 = 0.f;
    if (t < k) {  // (in front of the logits: their wait does not take these along)
        v0 = a.idx[row * k + t];
        x0 = load_elem(a.val, row * k + t, a.vdt);
    }
    const float w = a.drow ? a.drow[row] : 1.f;
    TdVec<T, CH> raw[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if ((i * 64 + t) * CH + CH <= V) raw[i] = *reinterpret_cast<const TdVec<T, CH>*>(z + (i * 64 + t) * CH);
    const int et = V - V % CH + t;  // what is left behind the last whole chunk, a logit a lane
    const T zt = et < V ? z[et] : T(0);
    float v[NCH][CH], m = -INFINITY, vt = -INFINITY;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int e0 = (i * 64 + t) * CH;
        if (e0 + CH <= V) {
            *reinterpret_cast<u32x4*>(rb + e0) = __builtin_bit_cast(u32x4, raw[i]);
#pragma unroll
            for (int e = 0; e < CH; ++e) v[i][e] = TdElem<DT>::get(raw[i].v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[i][e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < CH; ++e) m = fmaxf(m, v[i][e]);
    }
    if (et < V) {
        rb[et] = zt;
        vt = TdElem<DT>::get(zt);
        m = fmaxf(m, vt);
    }
    if (t == 0) sq[k] = 0.f;
    td_sync<1>();
    float tm = -INFINITY;
    for (int j = t; j < k; j += 64) {
        int c = j == t ? v0 : a.idx[row * k + j];
        const float x = (j == t ? x0 : load_elem(a.val, row * k + j, a.vdt)) * a.itau;
        if ((unsigned)c >= (unsigned)V) c = -1;
        sv[j] = (int16_t)c;
        slq[j] = x;
        if (c >= 0) {
            sz[j] = TdElem<DT>::get(rb[c]);
            tm = fmaxf(tm, x);
        }
    }
    m = td_reduce<1, true>(m, nullptr);
    tm = td_base(td_reduce<1, true>(tm, nullptr));
    const float mu = __builtin_isinf(m) ? 0.f : m;
    float s = 0.f, ts = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * 64 * CH < V)
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                v[i][e] = td_exp2(v[i][e], mu, a.c);
                s += v[i][e];
            }
    vt = td_exp2(vt, mu, a.c);
    s += vt;
    for (int j = t; j < k; j += 64)
        if (sv[j] >= 0) {
            const float lq = (slq[j] - tm) * kTdLog2e, q = __builtin_amdgcn_exp2f(lq);
            slq[j] = lq;
            sq[j] = q;
            ts += q;
        }
    s = td_reduce<1, false>(s, nullptr);
    ts = td_reduce<1, false>(ts, nullptr);
    const bool on = s != 0.f && ts != 0.f;
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s), its = 1.f / ts, lts = __builtin_amdgcn_logf(ts);
    td_sync<1>();  // every slot has read its logit: from here on the row says which slot names a class (k: none; of several, one of them)
    uint16_t* const own = reinterpret_cast<uint16_t*>(rb);
    const uint32_t none = (uint32_t)k * 0x10001u;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int e0 = (i * 64 + t) * CH;
        if (e0 + CH <= V)
#pragma unroll
            for (int e = 0; e < CH; e += 4) *reinterpret_cast<uint2*>(own + e0 + e) = uint2{none, none};
    }
    if (et < V) own[et] = (uint16_t)k;
    float sum = 0.f;
    for (int j = t; j < k; j += 64) {
        const float q = on && sv[j] >= 0 ? sq[j] * its : 0.f;
        sq[j] = q;
        if (q != 0.f) sum += q * ((slq[j] - lts + l2s) * kTdLn2 - (sz[j] - mu) * a.itau);  // (td_finish)
    }
    sum = td_reduce<1, false>(sum, nullptr);
    if (t == 0) td_row_out(a, row, on, sum);
    if (!dz) return;
    td_sync<1>();
    for (int j = t; j < k; j += 64)
        if (sv[j] >= 0) own[sv[j]] = (uint16_t)j;
    td_sync<1>();
    bool lost = false;  // another slot names this one's class
    for (int j = t; j < k; j += 64) lost = lost || (sv[j] >= 0 && own[sv[j]] != j);
    if (__ballot(lost)) {  // a class named twice takes the q of all of its slots, in their order
        for (int j = t; j < k; j += 64) {
            const int c = sv[j];
            if (c < 0 || own[c] != j) continue;
            float q = 0.f;
            for (int o = 0; o < k; ++o) q += sv[o] == c ? sq[o] : 0.f;
            sz[j] = q;
        }
        td_sync<1>();
        for (int j = t; j < k; j += 64)
            if (sv[j] >= 0 && own[sv[j]] == j) sq[j] = sz[j];
        td_sync<1>();
    }
    const float g = a.gs * w;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int e0 = (i * 64 + t) * CH;
        if (e0 + CH > V) continue;
        float o[CH];
#pragma unroll
        for (int e = 0; e < CH; ++e) o[e] = v[i][e] * inv;
#pragma unroll
        for (int e = 0; e < CH; e += 4) {
            const uint2 by = *reinterpret_cast<const uint2*>(own + e0 + e);
            if (((by.x ^ none) | (by.y ^ none)) != 0u) {
                o[e] -= sq[by.x & 0xffffu];
                o[e + 1] -= sq[by.x >> 16];
                o[e + 2] -= sq[by.y & 0xffffu];
                o[e + 3] -= sq[by.y >> 16];
            }
        }
#pragma unroll
        for (int e = 0; e < CH; ++e) o[e] = on ? o[e] * g : 0.f;
        td_put<GDT, CH>(dz + e0, o);
    }
    if (et < V) dz[et] = TdElem<GDT>::put(on ? (vt * inv - sq[own[et]]) * g : 0.f);
}

// V <= 32768: a row's logits in registers, up to NCH chunks of CH per thread, NW waves a row; loss, maximum and sum from one read. Bound by memory:
// 16800 x 8192 fp32 225 us = 4.9 TB/s, 4200 x 32768 223 us; shorter 16-bit rows by what a row waits for, so as few waves as hold one: bf16 with 2 and 4
// 20000 x 2100 57 and 79 us, x 3001 63 and 79, x 4096 75 and 79.
template <int DT, int GDT, int NW>
__global__ __launch_bounds__(NW * 64, NW == 16 ? 8 : 1) void td_wide_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int NT = NW * 64, CH = 16 / sizeof(T), NCH = 32 / CH;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ float scratch[16];
    const int t = (int)threadIdx.x, V = a.V;
    const int64_t row = a.row0 + blockIdx.x;
    const TdSlots slots(lds, a.k);
    const T* z;
    TG* dz;
    td_row(a, row, z, dz);

    float v[NCH][CH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int e0 = (i * NT + t) * CH;
        if (e0 + CH <= V) {
            const TdVec<T, CH> x = *reinterpret_cast<const TdVec<T, CH>*>(z + e0);
#pragma unroll
            for (int e = 0; e < CH; ++e) v[i][e] = TdElem<DT>::get(x.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[i][e] = -INFINITY;
            if (e0 < V)
#pragma unroll
                for (int e = 0; e < CH; ++e)
                    if (e0 + e < V) v[i][e] = TdElem<DT>::get(z[e0 + e]);
        }
    }
    bool on = td_teacher<DT, NW>(a, row, t, z, slots, scratch);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * NT * CH < V)
#pragma unroll
            for (int e = 0; e < CH; ++e) m = fmaxf(m, v[i][e]);
    m = td_reduce<NW, true>(m, scratch);
    const float mu = __builtin_isinf(m) ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * NT * CH < V)
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                v[i][e] = td_exp2(v[i][e], mu, a.c);
                s += v[i][e];
            }
    s = td_reduce<NW, false>(s, scratch);
    on = on && s != 0.f;
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s);
    const float g = a.gs * (a.drow ? a.drow[row] : 1.f), f = inv * g;
    if (dz) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int e0 = (i * NT + t) * CH;
            if (e0 >= V) continue;
            float o[CH];
#pragma unroll
            for (int e = 0; e < CH; ++e) o[e] = on ? v[i][e] * f : 0.f;
            if (e0 + CH <= V) td_put<GDT, CH>(dz + e0, o);
            else
#pragma unroll
                for (int e = 0; e < CH; ++e)
                    if (e0 + e < V) dz[e0 + e] = TdElem<GDT>::put(o[e]);
        }
    }
    td_sync<NW>();  // the slots are complete, the dense gradient is written: the named entries may follow
    td_finish<GDT, NW>(a, row, t, on, dz, mu, inv, l2s, g, slots, scratch);
}

// longer rows, as they are stored (16 waves a row, NCH chunks of 16 bytes a thread): two exponentials a logit instead of a second read.
// 8192 x 65536 bf16 415 us = 5.2 TB/s; NCH = 16 leaves one row a CU, whose loads and stores take turns: 4096 x 131072 bf16 487 us = 4.4 TB/s (walking over
// its rows, the next one's loads under this one's stores: 535). That form's time shows its instructions, so 16-bit rows take an exponent in one: z c - mu c,
// with the rounding of mu c (at most 1/2) taken back out of the sum (as (z - mu) c: 505 us, so 482; fp16 511 and 467). Where mu c is beyond 2^24 two 16-bit logits
// are the same or 2^12 and more apart, and a power of two that makes the product exact stands in for c.
template <int DT, int GDT, int NCH>
__global__ __launch_bounds__(1024, NCH <= 8 ? 8 : 4) void td_held_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int NW = 16, NT = 1024, CH = 16 / sizeof(T);
    constexpr uint32_t NINF = DT == CDET_F32 ? 0xff800000u : DT == CDET_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ float scratch[16];
    const int t = (int)threadIdx.x, V = a.V;
    const int64_t row = a.row0 + blockIdx.x;
    const TdSlots slots(lds, a.k);
    const T* z;
    TG* dz;
    td_row(a, row, z, dz);
    u32x4 v[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int e0 = (i * NT + t) * CH;
        v[i] = u32x4{NINF, NINF, NINF, NINF};
        if (e0 + CH <= V) {
            const TdVec<T, CH> x = *reinterpret_cast<const TdVec<T, CH>*>(z + e0);
            __builtin_memcpy(&v[i], &x, 16);
        }
    }
    const float vt = t < V % CH ? TdElem<DT>::get(z[V - V % CH + t]) : -INFINITY;  // what is left behind the last whole chunk: a logit a thread
    auto logit = [&](int i, int e) {
        if (DT == CDET_F32) return __uint_as_float(v[i][e]);
        return TdElem<DT>::get((T)(v[i][(e >> 1) & 3] >> (16 * (e & 1))));
    };
    // each pass unpacks the chunks anew: without this the compiler keeps 128 fp32 values a thread from the first pass on
    auto anew = [&](int i) { asm volatile("" : "+v"(v[i])); };
    const bool some = td_teacher<DT, NW>(a, row, t, z, slots, scratch);
    float m = vt;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * NT * CH < V) {
            anew(i);
#pragma unroll
            for (int e = 0; e < CH; ++e) m = fmaxf(m, logit(i, e));
        }
    m = td_reduce<NW, true>(m, scratch);
    const float mu = __builtin_isinf(m) ? 0.f : m;
    float c = a.c, muc = mu * c;
    if (DT != CDET_F32 && !(fabsf(muc) <= 16777216.f)) {
        c = __builtin_amdgcn_ldexpf(1.f, 23 - __builtin_amdgcn_frexp_expf(mu));
        muc = mu * c;
    }
    auto power = [&](float z, float mu, float muc) { return DT == CDET_F32 ? td_exp2(z, mu, c) : __builtin_amdgcn_exp2f(fmaf(z, c, -muc)); };
    float s = power(vt, mu, muc);
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * NT * CH < V) {
            anew(i);
#pragma unroll
            for (int e = 0; e < CH; ++e) s += power(logit(i, e), mu, muc);
        }
    s = td_reduce<NW, false>(s, scratch);
    const bool on = some && s != 0.f;
    const float g = a.gs * (a.drow ? a.drow[row] : 1.f), dense = g / s;
    if (DT != CDET_F32) s *= __builtin_amdgcn_exp2f(-fmaf(mu, c, -muc));
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s);
    if (dz) {
        float f = dense, mg = mu, mgc = muc;
        int u = t;
        asm volatile("" : "+v"(u));  // (addresses are computed anew: no register is kept for them)
        if (!on) {  // zeros, whatever the logits are
            f = mg = mgc = 0.f;
#pragma unroll
            for (int i = 0; i < NCH; ++i) v[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int e0 = (i * NT + u) * CH;
            if (i * NT * CH < V) {
                anew(i);
                float o[CH];
#pragma unroll
                for (int e = 0; e < CH; ++e) o[e] = power(logit(i, e), mg, mgc) * f;
                if (e0 + CH <= V) td_put<GDT, CH>(dz + e0, o);
            }
        }
        if (u < V % CH) dz[V - V % CH + u] = TdElem<GDT>::put(power(on ? vt : 0.f, mg, mgc) * f);
    }
    td_sync<NW>();
    td_finish<GDT, NW>(a, row, t, on, dz, mu, inv, l2s, g, slots, scratch);
}

// rows that do not fit the registers: one pass for a running maximum and sum, a second one for the gradient; 16 waves a row
// (1024 x 131072 fp32 315 us = 5.1 TB/s over its three passes)
template <int DT, int GDT>
__global__ __launch_bounds__(1024) void td_long_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int NW = 16, NT = 1024, CH = 16 / sizeof(T), U = 16 / CH;  // U chunks (16 logits) at a time
    extern __shared__ __attribute__((aligned(16))) float lds[];
    __shared__ float scratch[16];
    const int t = (int)threadIdx.x, V = a.V;
    const int64_t row = a.row0 + blockIdx.x;
    const TdSlots slots(lds, a.k);
    const T* z;
    TG* dz;
    td_row(a, row, z, dz);
    bool on = td_teacher<DT, NW>(a, row, t, z, slots, scratch);
    auto load = [&](int e0, float (&v)[CH]) {
        if (e0 + CH <= V) {
            const TdVec<T, CH> x = *reinterpret_cast<const TdVec<T, CH>*>(z + e0);
#pragma unroll
            for (int e = 0; e < CH; ++e) v[e] = TdElem<DT>::get(x.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < CH; ++e) v[e] = e0 + e < V ? TdElem<DT>::get(z[e0 + e]) : -INFINITY;
        }
    };
    float m = -INFINITY, s = 0.f;
    for (int b = 0; b < V; b += U * NT * CH) {
        float v[U][CH], mb = m;
#pragma unroll
        for (int u = 0; u < U; ++u) load(b + (u * NT + t) * CH, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < CH; ++e) mb = fmaxf(mb, v[u][e]);
        const float mu = __builtin_isinf(mb) ? 0.f : mb;
        s = s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f(((__builtin_isinf(m) ? 0.f : m) - mu) * a.c);
        m = mb;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < CH; ++e) s += __builtin_amdgcn_exp2f((v[u][e] - mu) * a.c);
    }
    const float all = td_reduce<NW, true>(m, scratch);
    const float mu = __builtin_isinf(all) ? 0.f : all;
    s = s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f(((__builtin_isinf(m) ? 0.f : m) - mu) * a.c);
    s = td_reduce<NW, false>(s, scratch);
    on = on && s != 0.f;
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s);
    const float g = a.gs * (a.drow ? a.drow[row] : 1.f), f = inv * g;
    if (dz) {
        for (int e0 = t * CH; e0 < V; e0 += NT * CH) {
            float v[CH];
            load(e0, v);
            float o[CH];
#pragma unroll
            for (int e = 0; e < CH; ++e) o[e] = on ? td_exp2(v[e], mu, a.c) * f : 0.f;
            if (e0 + CH <= V) td_put<GDT, CH>(dz + e0, o);
            else
#pragma unroll
                for (int e = 0; e < CH; ++e)
                    if (e0 + e < V) dz[e0 + e] = TdElem<GDT>::put(o[e]);
        }
    }
    td_sync<NW>();
    td_finish<GDT, NW>(a, row, t, on, dz, mu, inv, l2s, g, slots, scratch);
}

// N consecutive elements of which the first n exist, as fp32; the others `none`
template <int DT, int N>
__device__ __forceinline__ void td_get(const void* base, int64_t at, int n, float none, float (&v)[N]) {
    typedef typename TdElem<DT>::T T;
    const T* p = (const T*)base + at;
    if (n >= N) {
        const TdVec<T, N> u = *reinterpret_cast<const TdVec<T, N>*>(p);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = TdElem<DT>::get(u.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = e < n ? TdElem<DT>::get(p[e]) : none;
    }
}

// V <= L E, k <= L S: L lanes a row, E neighbouring classes and S slots a lane. A row's slots meet its classes in LDS: how far every class is below the maximum, and {q, 1} of the slot
// that named it last; as many owned classes as filled slots means that no class was named twice. Few elements a lane leave it bound by its instructions, so a
// lane takes four neighbours (6, 8 in longer rows) and, where k <= L, one slot: 268800 x 4 x 16 fp32, k = 16: 56 us = 5.1 TB/s, with a class and a slot a lane
// and 16 lanes a row 82; 268800 x 80 fp32, k = 10: 40 us (eight slots on each of two lanes took 1.6 times
// as long).
template <int DT, int GDT, int L, int E, int S>
__global__ __launch_bounds__(256) void td_narrow_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int ROWS = 256 / L, W = L * E + 4;  // (4: rows start in different banks)
    __shared__ __attribute__((aligned(16))) float s_z[ROWS][W];  // below the maximum
    __shared__ __attribute__((aligned(16))) float s_q[ROWS][2 * W];
    const int lane = (int)threadIdx.x & 63, l = (int)threadIdx.x & (L - 1), r = (int)threadIdx.x / L, V = a.V, k = a.k;
    const int64_t row = a.row0 + (int64_t)blockIdx.x * ROWS + r;
    const bool here = row < a.rows;
    const T* z;
    TG* dz;
    td_row(a, here ? row : 0, z, dz);
    const float w = a.drow && here ? a.drow[row] : 1.f;
    const int nv = here ? V - l * E : 0, nk = here ? k - l * S : 0;
    float v[E], tx[S];
    int ti[S];
    td_get<DT, E>(z, l * E, nv, -INFINITY, v);
    const int64_t at = (here ? row : 0) * k + l * S;
    if (a.vdt == CDET_F32) td_get<CDET_F32, S>(a.val, at, nk, 0.f, tx);
    else if (a.vdt == CDET_BF16) td_get<CDET_BF16, S>(a.val, at, nk, 0.f, tx);
    else td_get<CDET_F16, S>(a.val, at, nk, 0.f, tx);
    if (nk >= S) {
        const TdVec<int, S> u = *reinterpret_cast<const TdVec<int, S>*>(a.idx + at);
#pragma unroll
        for (int j = 0; j < S; ++j) ti[j] = u.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < S; ++j) ti[j] = j < nk ? a.idx[at + j] : -1;
    }
    float m = -INFINITY, tm = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
#pragma unroll
    for (int j = 0; j < S; ++j) {
        if ((unsigned)ti[j] >= (unsigned)V) ti[j] = -1;
        tx[j] = ti[j] >= 0 ? tx[j] * a.itau : -INFINITY;
        tm = fmaxf(tm, tx[j]);
    }
    m = td_lanes<L, true>(m);
    tm = td_base(td_lanes<L, true>(tm));
    const float mu = __builtin_isinf(m) ? 0.f : m;
    float s = 0.f, ts = 0.f, p[E], lq[S], q[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        lq[j] = (tx[j] - tm) * kTdLog2e;
        q[j] = ti[j] >= 0 ? __builtin_amdgcn_exp2f(lq[j]) : 0.f;
        ts += q[j];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] -= mu;
        p[e] = __builtin_amdgcn_exp2f(v[e] * a.c);
        s += p[e];
    }
    s = td_lanes<L, false>(s);
    ts = td_lanes<L, false>(ts);
    const bool on = s != 0.f && ts != 0.f;
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s), itq = 1.f / ts, lts = __builtin_amdgcn_logf(ts);
    float *below = s_z[r], *sq = s_q[r];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        *reinterpret_cast<float2*>(below + l * E + e) = float2{v[e], v[e + 1]};
        *reinterpret_cast<f32x4*>(sq + 2 * (l * E + e)) = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    td_sync<1>();  // (a row's lanes are in one wave)
    float sum = 0.f, more = 0.f;  // more: filled slots that own no class
#pragma unroll
    for (int j = 0; j < S; ++j)
        if (ti[j] >= 0) {
            q[j] *= itq;
            if (q[j] != 0.f) sum += q[j] * ((lq[j] - lts + l2s) * kTdLn2 - below[ti[j]] * a.itau);  // (td_finish)
            *reinterpret_cast<float2*>(sq + 2 * ti[j]) = float2{q[j], 1.f};
            more += 1.f;
        }
    td_sync<1>();
    sum = td_lanes<L, false>(sum);
    float qs[E];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const f32x4 o = *reinterpret_cast<const f32x4*>(sq + 2 * (l * E + e));
        qs[e] = o[0];
        qs[e + 1] = o[2];
        more -= o[1] + o[3];
    }
    more = td_lanes<L, false>(more);
    if (__ballot(more != 0.f)) {  // some class of these rows is named twice: add its slots up in their order
#pragma unroll
        for (int e = 0; e < E; ++e) qs[e] = 0.f;
        for (int j = 0; j * S < k; ++j) {
            const int src = (lane & (64 - L)) + j;
#pragma unroll
            for (int o = 0; o < S; ++o) {
                const int c = __shfl(ti[o], src) - l * E;
                const float qj = __shfl(q[o], src);
#pragma unroll
                for (int e = 0; e < E; ++e) qs[e] += c == e ? qj : 0.f;
            }
        }
    }
    if (!here) return;
    if (dz) {
        const float g = a.gs * w;
        float o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = on ? (p[e] * inv - qs[e]) * g : 0.f;
        if (nv >= E) td_put<GDT, E>(dz + l * E, o);
        else
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < nv) dz[l * E + e] = TdElem<GDT>::put(o[e]);
    }
    if (l == 0) td_row_out(a, row, on, sum);
}

template <int DT, int GDT>
static int td_launch_rows(const TdArgs& a, int64_t rows, hipStream_t s) {
    const size_t lds = (size_t)TdSlots::up(a.k) * 16;
#define CDET_NARROW(L, E)                                                                                          \
    do {                                                                                                           \
        const dim3 grid((unsigned)((rows + 256 / L - 1) / (256 / L)));                                           \
        if (a.k <= L) td_narrow_kernel<DT, GDT, L, E, 1><<<grid, dim3(256), 0, s>>>(a);                            \
        else td_narrow_kernel<DT, GDT, L, E, E><<<grid, dim3(256), 0, s>>>(a);                                     \
    } while (0)
    const int narrow = a.V > a.k ? a.V : a.k;
    if (narrow <= 16) CDET_NARROW(4, 4);
    else if (narrow <= 32) CDET_NARROW(8, 4);
    else if (narrow <= 64) CDET_NARROW(16, 4);
    else if (narrow <= 96) CDET_NARROW(16, 6);
    else if (narrow <= 128) CDET_NARROW(16, 8);
#undef CDET_NARROW
    else if (a.V <= 2048) {
        const dim3 grid((unsigned)((rows + 3) / 4));
        const size_t row = td_wave_lds<typename TdElem<DT>::T>(a.k, a.V);
        if (a.V <= 512) td_wave_kernel<DT, GDT, 8><<<grid, dim3(256), 4 * row, s>>>(a);
        else if (a.V <= 1024) td_wave_kernel<DT, GDT, 16><<<grid, dim3(256), 4 * row, s>>>(a);
        else td_wave_kernel<DT, GDT, 32><<<grid, dim3(256), 4 * row, s>>>(a);
    }
    else if (a.V <= 4096) td_wide_kernel<DT, GDT, 2><<<dim3((unsigned)rows), dim3(128), lds, s>>>(a);
    else if (a.V <= 8192) td_wide_kernel<DT, GDT, 4><<<dim3((unsigned)rows), dim3(256), lds, s>>>(a);
    else if (a.V <= 16384) td_wide_kernel<DT, GDT, 8><<<dim3((unsigned)rows), dim3(512), lds, s>>>(a);
    else if (a.V <= 32768) td_wide_kernel<DT, GDT, 16><<<dim3((unsigned)rows), dim3(1024), lds, s>>>(a);
    else if (DT != CDET_F32 && a.V <= 65536) td_held_kernel<DT, GDT, 8><<<dim3((unsigned)rows), dim3(1024), lds, s>>>(a);
    else if (a.V <= (DT == CDET_F32 ? 65536 : 131072)) td_held_kernel<DT, GDT, 16><<<dim3((unsigned)rows), dim3(1024), lds, s>>>(a);
    else td_long_kernel<DT, GDT><<<dim3((unsigned)rows), dim3(1024), lds, s>>>(a);
    CDET_LAUNCH_CHECK();
    return 0;
}

// (a launch of at most 2^31 threads)
template <int DT, int GDT>
static int td_launch(TdArgs a, hipStream_t s) {
    const int64_t most = a.V > 2048 ? 1 << 21 : 1 << 25;
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += most) {
        const int rc = td_launch_rows<DT, GDT>(a, a.rows - a.row0 < most ? a.rows - a.row0 : most, s);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace cdet

using namespace cdet;

extern "C" int cdet_topk_distill(const cdet_topk_distill_desc* d, const void* logits, const int32_t* idx, const void* val, const float* drow, float* loss, void* dlogits,
                                 void* stream) {
    CDET_CHECK_ARG(d, "cdet_topk_distill: no descriptor");
    auto flt = [](int t) { return t == CDET_F32 || t == CDET_BF16 || t == CDET_F16; };
    CDET_CHECK_ARG(flt(d->dtype) && flt(d->val_dtype) && (d->grad_dtype == d->dtype || d->grad_dtype == CDET_F32),
                   "cdet_topk_distill: types %d / %d must be fp32, bf16 or fp16, the gradient's (%d) the logits' or fp32", d->dtype, d->val_dtype, d->grad_dtype);
    CDET_CHECK_ARG(d->P >= 0 && d->G >= 1 && d->V >= 1 && d->V <= (1 << 24) && (int64_t)d->P * d->G < ((int64_t)1 << 31), "cdet_topk_distill: P %d, G %d, V %d", d->P,
                   d->G, d->V);
    CDET_CHECK_ARG(d->k >= 1 && d->k <= 512, "cdet_topk_distill: k = %d (1 .. 512)", d->k);
    CDET_CHECK_ARG(d->tau >= 1e-18f && d->tau <= 1e18f, "cdet_topk_distill: tau %g (1e-18 .. 1e18)", d->tau);  // (1 / tau and tau^2 are fp32 numbers)
    CDET_CHECK_ARG(d->ld >= 0, "cdet_topk_distill: negative pitch");
    if (d->P == 0) return 0;
    CDET_CHECK_ARG(logits && idx && val && loss, "cdet_topk_distill: logits, idx, val and loss must be given");
    CDET_CHECK_ARG(!dlogits || d->grad_ld >= (int64_t)d->G * d->V, "cdet_topk_distill: the gradient's pitch %lld is below G * V", (long long)d->grad_ld);
    CDET_CHECK_ARG(dlogits != logits || (d->grad_dtype == d->dtype && d->grad_ld == d->ld), "cdet_topk_distill: in place needs the logits' type and pitch");
    const int es = elem_size(d->dtype), gs = elem_size(d->grad_dtype);
    CDET_CHECK_ARG(((uintptr_t)logits % es) == 0 && ((uintptr_t)dlogits % gs) == 0, "cdet_topk_distill: logits / dlogits must be aligned to their elements");
    if (dlogits && dlogits != logits) {  // beside the logits (another slice of their map, say), not half over them: rows are read while others are written
        const uintptr_t z = (uintptr_t)logits, g = (uintptr_t)dlogits;
        const int64_t zp = d->ld * es, gp = d->grad_ld * gs, zw = (int64_t)d->G * d->V * es, gw = (int64_t)d->G * d->V * gs;
        bool apart = g >= z + (uintptr_t)((d->P - 1) * zp + zw) || z >= g + (uintptr_t)((d->P - 1) * gp + gw);
        if (!apart && zp == gp) {
            const int64_t in = ((int64_t)(g - z) % zp + zp) % zp;  // where in a pixel of the logits the gradient starts
            apart = in >= zw && in + gw <= zp;
        }
        CDET_CHECK_ARG(apart, "cdet_topk_distill: the gradient overlaps the logits without being in their place");
    }
    TdArgs a;
    a.z = logits;
    a.dz = dlogits;
    a.idx = idx;
    a.val = val;
    a.drow = drow;
    a.loss = loss;
    a.part = d->part;
    a.ld = d->ld;
    a.gld = d->grad_ld;
    a.rows = (int64_t)d->P * d->G;
    a.G = d->G;
    a.V = d->V;
    a.k = d->k;
    a.vdt = d->val_dtype;
    a.c = kTdLog2e / d->tau;
    a.itau = 1.f / d->tau;
    a.tau2 = d->tau * d->tau;
    a.gs = d->grad_scale * d->tau;
    hipStream_t s = (hipStream_t)stream;
    if (d->dtype == CDET_F32) return td_launch<CDET_F32, CDET_F32>(a, s);
    if (d->dtype == CDET_BF16) return d->grad_dtype == CDET_F32 ? td_launch<CDET_BF16, CDET_F32>(a, s) : td_launch<CDET_BF16, CDET_BF16>(a, s);
    return d->grad_dtype == CDET_F32 ? td_launch<CDET_F16, CDET_F32>(a, s) : td_launch<CDET_F16, CDET_F16>(a, s);
}
