// Distillation from a teacher's top k logits on logits that are in memory: loss and gradient of every row in one launch.
//   p = softmax(z / tau) over the row's V logits, q = softmax of the teacher's filled slots / tau
//   loss = tau^2 sum_j q_j (log q_j - log p[idx_j]),   dz_v = drow * grad_scale * tau * (p_v - sum_{j: idx_j == v} q_j)
// Bound by memory: logits once in, gradient once out. A row of up to 32768 logits stays in the registers of its 1, 4 or 16 waves (td_wide_kernel), so the
// maximum, the sum and the gradient are taken from one read; a longer row is read again for its gradient (td_long_kernel: the second read comes out of
// the 256 MiB cache). The gradient is written dense and then, behind a barrier, the k named entries are written again with their q. Rows of at most 64
// logits (box distributions) take 16 lanes each and put q together in LDS first (td_narrow_kernel). p is exp2((z - max) c) / sum: its error does not
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
    int64_t ld, gld;
    int64_t rows;
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

// sums / maxima over the workgroup's waves (NW = 1: inside the wave), the same value in every thread, in a fixed order
template <int NW, bool MAX>
__device__ __forceinline__ float td_reduce(float v, float* scratch) {
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const float u = __shfl_xor(v, o);
        v = MAX ? fmaxf(v, u) : v + u;
    }
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

// a row's teacher in LDS: class (-1: an empty slot), q, log q, and the student's logit there (taken before the gradient may overwrite it)
struct TdSlots {
    float *q, *lq, *z;
    int* v;
    __device__ TdSlots(float* lds, int k) : q(lds), lq(lds + k), z(lds + 2 * k), v(reinterpret_cast<int*>(lds + 3 * k)) {}
};
// fills it; t = thread of the row. False: no filled slot, or nothing but -inf in them
template <int DT, int NW>
__device__ __forceinline__ bool td_teacher(const TdArgs& a, int64_t row, int t, const typename TdElem<DT>::T* z, TdSlots s, float* scratch) {
    constexpr int NT = NW * 64;
    float m = -INFINITY;
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
    m = td_reduce<NW, true>(m, scratch);
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
    return m != -INFINITY;
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
        const float e2 = (s.z[j] - mu) * a.c;
        if (q != 0.f) sum += q * (s.lq[j] - (e2 - l2s) * kTdLn2);
        if (!dz) continue;
        bool first = true;
        for (int o = 0; o < a.k; ++o) {
            const bool same = s.v[o] == v;
            first = first && !(same && o < j);
            q += same && o > j ? s.q[o] : 0.f;
        }
        if (first) dz[v] = TdElem<GDT>::put((__builtin_amdgcn_exp2f(e2) * inv - q) * g);
    }
    sum = td_reduce<NW, false>(sum, scratch);
    if (t == 0) a.loss[row] = on ? sum * a.tau2 : 0.f;
}

template <typename T, typename TG>
__device__ __forceinline__ void td_row(const TdArgs& a, int64_t row, const T*& z, TG*& dz) {
    const int64_t px = row / a.G, gr = row - px * a.G;
    z = (const T*)a.z + px * a.ld + gr * a.V;
    dz = a.dz ? (TG*)a.dz + px * a.gld + gr * a.V : nullptr;
}

// a row's logits in registers: up to NCH chunks of CH per thread, NW waves a row (NW = 1: four rows a workgroup)
template <int DT, int GDT, int NW>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void td_wide_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int NT = NW * 64, CH = 16 / sizeof(T), NCH = 32 / CH;
    extern __shared__ float lds[];
    __shared__ float scratch[16];
    const int sub = NW == 1 ? (int)threadIdx.x >> 6 : 0, t = (int)threadIdx.x & (NT - 1), V = a.V;
    const int64_t row = (int64_t)blockIdx.x * (NW == 1 ? 4 : 1) + sub;
    if (row >= a.rows) return;  // (NW == 1: whole waves, and no barrier of the workgroup follows)
    const TdSlots slots(lds + sub * 4 * a.k, a.k);
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
    on = on && m != -INFINITY;
    const float mu = __builtin_isinf(m) ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
        if (i * NT * CH < V)
#pragma unroll
            for (int e = 0; e < CH; ++e) {
                v[i][e] = __builtin_amdgcn_exp2f((v[i][e] - mu) * a.c);
                s += v[i][e];
            }
    s = td_reduce<NW, false>(s, scratch);
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s);
    const float g = a.gs * (a.drow ? a.drow[row] : 1.f);
    if (dz) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int e0 = (i * NT + t) * CH;
            if (e0 >= V) continue;
            TdVec<TG, CH> o;
#pragma unroll
            for (int e = 0; e < CH; ++e) o.v[e] = TdElem<GDT>::put(on ? v[i][e] * inv * g : 0.f);
            if (e0 + CH <= V) *reinterpret_cast<TdVec<TG, CH>*>(dz + e0) = o;
            else
#pragma unroll
                for (int e = 0; e < CH; ++e)
                    if (e0 + e < V) dz[e0 + e] = o.v[e];
        }
    }
    td_sync<NW>();  // the slots are complete, the dense gradient is written: the named entries may follow
    td_finish<GDT, NW>(a, row, t, on, dz, mu, inv, l2s, g, slots, scratch);
}

// rows that do not fit the registers: one pass for a running maximum and sum, a second one for the gradient; 16 waves a row
template <int DT, int GDT>
__global__ __launch_bounds__(1024) void td_long_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int NW = 16, NT = 1024, CH = 16 / sizeof(T), U = 16 / CH;  // U chunks (16 logits) at a time
    extern __shared__ float lds[];
    __shared__ float scratch[16];
    const int t = (int)threadIdx.x, V = a.V;
    const int64_t row = blockIdx.x;
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
    on = on && all != -INFINITY;
    const float mu = __builtin_isinf(all) ? 0.f : all;
    s = s == 0.f ? 0.f : s * __builtin_amdgcn_exp2f(((__builtin_isinf(m) ? 0.f : m) - mu) * a.c);
    s = td_reduce<NW, false>(s, scratch);
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s);
    const float g = a.gs * (a.drow ? a.drow[row] : 1.f);
    if (dz) {
        for (int e0 = t * CH; e0 < V; e0 += NT * CH) {
            float v[CH];
            load(e0, v);
            TdVec<TG, CH> o;
#pragma unroll
            for (int e = 0; e < CH; ++e) o.v[e] = TdElem<GDT>::put(on ? __builtin_amdgcn_exp2f((v[e] - mu) * a.c) * inv * g : 0.f);
            if (e0 + CH <= V) *reinterpret_cast<TdVec<TG, CH>*>(dz + e0) = o;
            else
#pragma unroll
                for (int e = 0; e < CH; ++e)
                    if (e0 + e < V) dz[e0 + e] = o.v[e];
        }
    }
    td_sync<NW>();
    td_finish<GDT, NW>(a, row, t, on, dz, mu, inv, l2s, g, slots, scratch);
}

// V <= 64, k <= 64: 16 lanes a row, 16 rows a workgroup. Per row in LDS: the logits' log p, the q of every class, who named a class last
template <int DT, int GDT>
__global__ __launch_bounds__(256) void td_narrow_kernel(const TdArgs a) {
    typedef typename TdElem<DT>::T T;
    typedef typename TdElem<GDT>::T TG;
    constexpr int E = 4;
    __shared__ float s_lp[16][64], s_q[16][64];
    __shared__ int s_own[16][64];
    const int l = (int)threadIdx.x & 15, r = (int)threadIdx.x >> 4, V = a.V, k = a.k;
    const int64_t row = (int64_t)blockIdx.x * 16 + r;
    const bool here = row < a.rows;
    const T* z;
    TG* dz;
    td_row(a, here ? row : 0, z, dz);
    auto gmax = [](float v) {
#pragma unroll
        for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
        return v;
    };
    auto gsum = [](float v) {
#pragma unroll
        for (int o = 8; o; o >>= 1) v += __shfl_xor(v, o);
        return v;
    };
    float v[E], tx[E];
    int ti[E];
    float m = -INFINITY, tm = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = here && e * 16 + l < V ? TdElem<DT>::get(z[e * 16 + l]) : -INFINITY;
        const int j = e * 16 + l;
        ti[e] = -1;
        tx[e] = -INFINITY;
        if (here && j < k) {
            const int c = a.idx[row * k + j];
            ti[e] = (unsigned)c < (unsigned)V ? c : -1;
            if (ti[e] >= 0) tx[e] = load_elem(a.val, row * k + j, a.vdt) * a.itau;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        m = fmaxf(m, v[e]);
        tm = fmaxf(tm, tx[e]);
    }
    m = gmax(m);
    tm = gmax(tm);
    const float mu = __builtin_isinf(m) ? 0.f : m;
    const bool on = tm != -INFINITY && m != -INFINITY;
    float s = 0.f, ts = 0.f;
    float p[E], lq[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        lq[e] = tx[e] - tm;
        if (ti[e] >= 0) ts += expf(lq[e]);
        v[e] = (v[e] - mu) * a.c;
        p[e] = __builtin_amdgcn_exp2f(v[e]);
        s += p[e];
    }
    s = gsum(s);
    ts = gsum(ts);
    const float inv = 1.f / s, l2s = __builtin_amdgcn_logf(s), lts = logf(ts);
    float q[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        lq[e] -= lts;
        q[e] = ti[e] >= 0 ? expf(lq[e]) : 0.f;
        if (e * 16 < V) {
            s_lp[r][e * 16 + l] = (v[e] - l2s) * kTdLn2;
            s_q[r][e * 16 + l] = 0.f;
        }
    }
    td_sync<1>();  // (a row's 16 lanes are in one wave)
    float sum = 0.f;
    bool twice = false;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (ti[e] >= 0) {
            if (q[e] != 0.f) sum += q[e] * (lq[e] - s_lp[r][ti[e]]);
            s_own[r][ti[e]] = e * 16 + l;
            s_q[r][ti[e]] = q[e];
        }
    td_sync<1>();
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (ti[e] >= 0 && s_own[r][ti[e]] != e * 16 + l) twice = true;
    sum = gsum(sum);
    float qs[E];
#pragma unroll
    for (int e = 0; e < E; ++e) qs[e] = e * 16 < V ? s_q[r][e * 16 + l] : 0.f;
    if (__ballot(twice)) {  // some class of these rows is named twice: add its slots up in their order
#pragma unroll
        for (int e = 0; e < E; ++e) qs[e] = 0.f;
        for (int j = 0; j < k; ++j) {
            const int src = ((int)threadIdx.x & 48) + (j & 15);
            int c = -1;
            float qj = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int ce = __shfl(ti[e], src);
                const float qe = __shfl(q[e], src);
                if (j >> 4 == e) {
                    c = ce;
                    qj = qe;
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) qs[e] += c == e * 16 + l ? qj : 0.f;
        }
    }
    if (!here) return;
    const float g = a.gs * (a.drow ? a.drow[row] : 1.f);
    if (dz) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e * 16 + l < V) dz[e * 16 + l] = TdElem<GDT>::put(on ? (p[e] * inv - qs[e]) * g : 0.f);
    }
    if (l == 0) a.loss[row] = on ? sum * a.tau2 : 0.f;
}

template <int DT, int GDT>
static int td_launch(const TdArgs& a, hipStream_t s) {
    const size_t lds = (size_t)a.k * 16;
    if (a.V <= 64 && a.k <= 64) td_narrow_kernel<DT, GDT><<<dim3((unsigned)((a.rows + 15) / 16)), dim3(256), 0, s>>>(a);
    else if (a.V <= 2048) td_wide_kernel<DT, GDT, 1><<<dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 4 * lds, s>>>(a);
    else if (a.V <= 8192) td_wide_kernel<DT, GDT, 4><<<dim3((unsigned)a.rows), dim3(256), lds, s>>>(a);
    else if (a.V <= 32768) td_wide_kernel<DT, GDT, 16><<<dim3((unsigned)a.rows), dim3(1024), lds, s>>>(a);
    else td_long_kernel<DT, GDT><<<dim3((unsigned)a.rows), dim3(1024), lds, s>>>(a);
    CDET_LAUNCH_CHECK();
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
    CDET_CHECK_ARG(d->tau > 0.f && d->tau < INFINITY, "cdet_topk_distill: tau %g must be positive", d->tau);
    CDET_CHECK_ARG(d->ld >= 0, "cdet_topk_distill: negative pitch");
    if (d->P == 0) return 0;
    CDET_CHECK_ARG(logits && idx && val && loss, "cdet_topk_distill: logits, idx, val and loss must be given");
    CDET_CHECK_ARG(!dlogits || d->grad_ld >= (int64_t)d->G * d->V, "cdet_topk_distill: the gradient's pitch %lld is below G * V", (long long)d->grad_ld);
    CDET_CHECK_ARG(dlogits != logits || (d->grad_dtype == d->dtype && d->grad_ld == d->ld), "cdet_topk_distill: in place needs the logits' type and pitch");
    const int es = elem_size(d->dtype), gs = elem_size(d->grad_dtype);
    CDET_CHECK_ARG(((uintptr_t)logits % es) == 0 && ((uintptr_t)dlogits % gs) == 0, "cdet_topk_distill: logits / dlogits must be aligned to their elements");
    TdArgs a;
    a.z = logits;
    a.dz = dlogits;
    a.idx = idx;
    a.val = val;
    a.drow = drow;
    a.loss = loss;
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
