// Losses of a linear class projection over a long class list, logits never in memory:
//   z[r][v] = scale * <x_r, w_v> + offset[v]          x [N, d], w [V, d], 16-bit; everything below in fp32
//   cross entropy   loss_r = lse_r - z[r][label_r],                       dz[r][v] = g_r (p[r][v] - [v == label_r])
//   distillation    loss_r = tau^2 sum_j q_rj (log q_rj - log p[r][idx_rj]), dz[r][v] = g_r tau (p[r][v] - sum_{j: idx_rj == v} q_rj)
// with p = softmax(z / tau) and q the softmax of the teacher's k logits / tau. dx = scale * dz w, dw = scale * dz^T x.
//
// Forward: one matrix product whose epilogue keeps, per row and per 128 (64) classes, the running maximum and the sum of exponentials; a second launch
// joins those pairs per row in a fixed order. Backward: per piece of the class list the product is computed again, its epilogue turns the logits
// into dz (16-bit, one [N, piece] buffer), and one launch computes the piece's dw and adds the piece to dx. dz is relative to the largest row gradient
// (class_prep_kernel): p of a 10^5-class list times 1 / N is far below fp16's smallest number. That rounding is the price of multiplying dz on the matrix
// cores once: relative to 64 bits dx and dw are off by 0.0018 - 0.0024 (bf16) and 0.00026 - 0.00029 (fp16), by 0.0017 and 0.00021 with dz in fp32, whose rounding
// of the results alone remains; dz as two 16-bit numbers would double both gradient products, half of a training pass (up to 64 rows they are not what counts).
//
// One product for all three (Pipe): an 8-wave workgroup, 256 x 256 outputs, K in steps of 32 through a ring of four LDS stages filled by LDS-DMA. The two
// halves of the workgroup run half a step apart: while one multiplies, the other reads its fragments. What bounds it is the chip's power: 4096 x 4096 x 8192
// runs at 1230 - 1250 TF/s on random bf16 numbers and at 1740 on zeros (a library's product on the same random numbers: 1300). Small problems take 128 x 128 tiles of
// 4 waves (Quad), where a workgroup's own latency counts; the backward of at most 128 rows has a form of its own (class_few_kernel).
// Operand "A" (fragment rows) is what must come out contiguous: a lane ends up with four consecutive A rows of one B row. So A = classes in the first
// product (a lane holds classes of ONE row of x: the softmax statistics are sums inside the lane), A = features in the other two. An operand whose
// memory runs along the output index instead of K is staged as it lies and transposed by ds_read_b64_tr_b16 on the way to the registers.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.h"

namespace cdet {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(2))) float cf32x2;
typedef __attribute__((ext_vector_type(2))) __bf16 cbf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 cf16x2;

constexpr int LBK = 32;                   // K elements per step
constexpr int LRING = 4;                  // LDS stages
constexpr unsigned LSENT = 0xE0000000u;   // offset beyond every buffer: the DMA writes zeros
constexpr int LCAP = (int)0xD0000000u;    // extent of every buffer descriptor (offsets are at most 256 rows or 32 rows of < 4 M elements)
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// bit masks (which rows take part, which classes are not left out), read through the scalar cache: they do not count with the DMA
typedef const __attribute__((address_space(4))) uint32_t* mask_t;
__device__ __forceinline__ mask_t as_mask(const uint32_t* p) { return (mask_t)(uintptr_t)p; }

// a class's offset in log2 units; -inf leaves the class out, in every form: an offset of -inf, or a mask near fp32's lowest number
__device__ __forceinline__ float class_offset(float off, float coff) { return off < -2.3e38f ? -INFINITY : off * coff; }

template <int DT>
__device__ __forceinline__ f32x16 lmfma(const u32x4& a, const u32x4& b, const f32x16& c) {
    if (DT == CDET_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t lpack2(float a, float b) {  // round to nearest even
    if (DT == CDET_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(cf32x2{a, b}, cbf16x2));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(cf32x2{a, b}, cf16x2));
}
__device__ __forceinline__ int xcd_order(int b, int n) {  // consecutive logical ids run on one XCD (bijective)
    const int xcd = b & 7, q = n >> 3, r = n & 7, j = b >> 3;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + j;
}

// The staged stream of a workgroup's tiles and the multiplications on it. acc[mt][nt] = A B^T over K (any K; K % 8 == 0 for K-contiguous operands); C row of
// register i: grp * MT*32 + mt*32 + 8*(i>>2) + 4*(lane>>5) + (i&3), C column: wave * NT*32 + nt*32 + (lane&31). The stream runs three stages ahead of the
// multiplications, across the end of a tile: what `next` opens is fetched while the last tile is finished and its results are stored.
// WALK = false: one tile only, without the branches of the crossing. KM (ATR, no walk): open() takes a bit per k; what takes no part is not read from A.
template <int DT, int MT, int NT, bool ATR, bool BTR, bool WALK, bool KM>
struct Pipe {
    static constexpr int ABYTES = MT * 64 * 64, BBYTES = NT * 128 * 64, STAGE = ABYTES + BBYTES;
    static constexpr int NA = MT / 2, NB = NT, NPW = NA + NB;  // DMA instructions (1 KiB) of a wave per step
    unsigned char* smem;
    int lane, wave8, grp, wave, aoff, boff;
    unsigned va[NA], vb[NB];
    int ka[NA], kb[NB];  // the lane's first k of the piece
    const uint16_t *ap, *bp;
    int64_t astep, bstep;
    int krem;            // K of the opened tile left to be fetched
    int fslot, rslot;    // stages to be written / read next (byte offsets)
    int sure;            // memory phases whose next stage is known to be there
    mask_t km;           // KM: word of the fourth stage from now; w[]: of the next three
    uint32_t w[3];

    __device__ __forceinline__ void init(unsigned char* s, int64_t a_ld, int64_t b_ld) {
        smem = s;
        const int tid = (int)threadIdx.x;
        lane = tid & 63;
        wave8 = __builtin_amdgcn_readfirstlane(tid >> 6);
        grp = wave8 >> 2;
        wave = wave8 & 3;
        const int l31 = lane & 31, h = lane >> 5;
        // DMA sources. K-contiguous: piece `id` = rows 16 id .. +15, four lanes (64 B) a row, 16-byte slot s of row r stored at s ^ ((r >> 2) & 3): the 16
        // lanes that one ds_read_b128 cycle serves then cover the 16 slots of 256 bytes. Transposed: piece `id` = 64 rows x 8 k, eight lanes (128 B) a k;
        // slot s of k stored at s ^ (4 * ((k >> 1) & 1)): the four k of a transpose read, and its two 16-row halves, fall into different banks.
#pragma unroll
        for (int i = 0; i < NA; ++i) va[i] = ATR ? (unsigned)(k_of(ATR, i) * a_ld + row_of(ATR, i)) * 2u : (unsigned)(row_of(ATR, i) * a_ld + k_of(ATR, i)) * 2u;
#pragma unroll
        for (int i = 0; i < NB; ++i) vb[i] = BTR ? (unsigned)(k_of(BTR, i) * b_ld + row_of(BTR, i)) * 2u : (unsigned)(row_of(BTR, i) * b_ld + k_of(BTR, i)) * 2u;
        astep = ATR ? LBK * a_ld : LBK;
        bstep = BTR ? LBK * b_ld : LBK;
        const int trl = (8 * h + ((lane & 15) >> 2)) * 128 + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ (((lane >> 3) & 1) << 2)) << 4) + (lane & 1) * 8;
        const int nrl = l31 * 64 + ((h ^ ((l31 >> 2) & 3)) << 4);
        aoff = ATR ? trl + grp * (MT / 2) * 4096 : nrl + grp * MT * 2048;
        boff = ABYTES + (BTR ? (trl ^ (((wave * NT) & 1) << 6)) + ((wave * NT) >> 1) * 4096 : nrl + wave * NT * 2048);
        fslot = rslot = sure = 0;
    }
    __device__ __forceinline__ int k_of(bool tr, int i) const {
        const int id = wave8 + 8 * i;
        return tr ? 8 * (id & 3) + (lane >> 3) : 8 * ((lane & 3) ^ ((lane >> 4) & 3));
    }
    __device__ __forceinline__ int row_of(bool tr, int i) const {
        const int id = wave8 + 8 * i;
        return tr ? (id >> 2) * 64 + 8 * ((lane & 7) ^ (((lane >> 4) & 1) << 2)) : 16 * id + (lane >> 2);
    }
    // the tile that is fetched from now on (rows beyond a_rows / b_rows, and everything beyond K, read as zero; a_rows 0: nothing is read)
    __device__ __forceinline__ void open(const uint16_t* a, int a_rows, const uint16_t* b, int b_rows, int K, const uint32_t* k_mask = nullptr) {
#pragma unroll
        for (int i = 0; i < NA; ++i) ka[i] = KM ? (row_of(ATR, i) < a_rows ? 1 << k_of(ATR, i) : 0) : row_of(ATR, i) < a_rows ? k_of(ATR, i) : 0x40000000;
#pragma unroll
        for (int i = 0; i < NB; ++i) kb[i] = row_of(BTR, i) < b_rows ? k_of(BTR, i) : 0x40000000;
        ap = a;
        bp = b;
        krem = K;
        if (KM) {
            km = as_mask(k_mask);
            w[0] = km[0];
            w[1] = km[1];
            w[2] = km[2];
            km += 3;
        }
    }
    __device__ __forceinline__ uint32_t read_word() { return KM ? *km++ : 0u; }  // (the masks are longer than their numbers by what is read ahead)
    __device__ __forceinline__ void push_word(uint32_t word) {
        if (!KM) return;
        w[0] = w[1];
        w[1] = w[2];
        w[2] = word;
    }
    template <class Next>
    __device__ __forceinline__ void fetch(Next&& next) {
        if (WALK && krem <= 0) next();
        const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)ap, 0, LCAP, 0x00020000);
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void*)bp, 0, LCAP, 0x00020000);
        unsigned char* dst = smem + fslot + wave8 * 1024;
        const int word = KM ? (int)(krem >= LBK ? w[0] : krem > 0 ? w[0] & ((1u << krem) - 1) : 0u) : 0;
#pragma unroll
        for (int i = 0; i < NA; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(dst + i * 8192), 16,
                                                     (int)((KM ? (ka[i] & word) != 0 : ka[i] < krem) ? va[i] : LSENT), 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NB; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void*)(dst + ABYTES + i * 8192), 16, (int)(kb[i] < krem ? vb[i] : LSENT), 0, 0, 0);
        ap += astep;
        bp += bstep;
        krem -= LBK;
        fslot = fslot + STAGE == LRING * STAGE ? 0 : fslot + STAGE;
    }
    template <class Next>
    __device__ __forceinline__ void prime(Next&& next) {
        for (int f = 0; f < 3; ++f) {
            fetch(next);
            push_word(read_word());
        }
    }
    __device__ __forceinline__ void start() {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * NPW) : "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ u32x4 frag_n(int base, int t, int kk) const { return *reinterpret_cast<const u32x4*>(smem + ((base + t * 2048) ^ (kk << 5))); }
    // transpose reads are asm: in front of the builtin the compiler waits for every DMA in flight. Their registers become values behind the phase's own wait;
    // that the compiler moves none of them before it is checked in the build's assembly (tests/test_class_loss_registers_cpu.py)
    __device__ __forceinline__ void frag_t(int base, int t, int kk, u32x2& lo, u32x2& hi) const {
        const int o = (int)(unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem + (((base + (t >> 1) * 4096) ^ ((t & 1) << 6)) + kk * 2048);
        asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(lo) : "v"(o));
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:512" : "=v"(hi) : "v"(o));
    }

    // One tile. A step of a wave is a memory phase (fragment reads, one stage fetched) and a compute phase, each closed by a barrier; waves 4-7 run one phase
    // behind waves 0-3. Every wave returns past its last read of the tile's last stage, whose slot, free(), nobody touches before the next fetch().
    template <class Next>
    __device__ __forceinline__ void run(int steps, f32x16 (&acc)[MT][NT], Next&& next) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        if (grp == 1) {
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int st = 0; st < steps; ++st) {
            u32x4 a[2][MT], b[2][NT];
            u32x2 al[2][MT], ah[2][MT], bl[2][NT], bh[2][NT];
            if (KM) asm volatile("" : "+s"(w[0]), "+s"(w[1]), "+s"(w[2]));
            const uint32_t word = read_word();
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    if (BTR) frag_t(rslot + boff, i, kk, bl[kk][i], bh[kk][i]);
                    else b[kk][i] = frag_n(rslot + boff, i, kk);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    if (ATR) frag_t(rslot + aoff, i, kk, al[kk][i], ah[kk][i]);
                    else a[kk][i] = frag_n(rslot + aoff, i, kk);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            // stage st + 3 goes where stage st - 1 was: its last reader, the other half in ITS memory phase of step st - 1, waited for its reads before
            // the barrier that opened this phase
            fetch(next);
            rslot = rslot + STAGE == LRING * STAGE ? 0 : rslot + STAGE;
            __builtin_amdgcn_sched_barrier(0);
            // stage st + 1 has landed for this wave (two stages stay in flight); the fragments are in registers
            if (WALK && sure > 0) {
                --sure;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            } else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * NPW) : "memory");
            push_word(word);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                if (ATR) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        asm volatile("" : "+v"(al[kk][i]), "+v"(ah[kk][i]));
                        a[kk][i] = u32x4{al[kk][i][0], al[kk][i][1], ah[kk][i][0], ah[kk][i][1]};
                    }
                }
                if (BTR) {
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        asm volatile("" : "+v"(bl[kk][i]), "+v"(bh[kk][i]));
                        b[kk][i] = u32x4{bl[kk][i][0], bl[kk][i][1], bh[kk][i][0], bh[kk][i][1]};
                    }
                }
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = lmfma<DT>(a[kk][i], b[kk][j], acc[i][j]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (st + 1 < steps) {
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (grp == 0) {  // releases the other half into its last multiplication
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __device__ __forceinline__ unsigned char* free_slot() const { return smem + (rslot == 0 ? (LRING - 1) * STAGE : rslot - STAGE); }
    // before the tile's stores (they count like loads): the three stages in flight land, so that the next two memory phases need not wait behind the stores
    __device__ __forceinline__ void settle() {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        sure = 2;
    }
    __device__ __forceinline__ void sync() {  // every wave is done with free_slot(), and with its share of the stages in flight
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void drain() {  // after the last tile: the (empty) fetches in flight write zeros into the ring; then the LDS is free
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
};

// The small tile, for launches that leave most of the chip idle: what counts is how long ONE workgroup takes for a step. Four waves (2 x 2) of MT x NT row
// tiles, no phases: a wave multiplies one half of a step while it reads the next half's fragments, one barrier a step, RING - 1 stages ahead. (As phases of
// 8 waves, like the large tile, the two products of 997 x 1201 x 320's gradients took 16.1 us, so 13.7; a deeper ring does not help.) Same interface as Pipe; column = wave * NT*32 + nt*32 + (lane&31),
// wave = 0, 1; run() leaves the LDS free. Rows and classes that take no part are not read: open() takes a bit per row of B, and (KM) per k of A -- a launch
// less than a copy of x without them, which the large tile is given instead: in its loop the test costs 2 - 3 % of a product, more than the copy of x does;
// for w (KEPT, below) it is the copy that costs more.
template <int DT, int MT, int NT, bool ATR, bool BTR, int RING, bool KM>
struct Quad {
    static constexpr int ABYTES = MT * 64 * 64, BBYTES = NT * 64 * 64, STAGE = ABYTES + BBYTES;
    static constexpr int NA = MT, NB = NT, NPW = NA + NB;
    unsigned char* smem;
    int lane, wave8, grp, wave, aoff, boff;
    unsigned va[NA], vb[NB];
    int ka[NA], kb[NB];
    const uint16_t *ap, *bp;
    int64_t astep, bstep;
    int krem, fslot;
    mask_t km;     // k mask: word of the fourth stage from now; w[]: of the next three
    uint32_t w[3];

    __device__ __forceinline__ int k_of(bool tr, int i) const {
        const int id = wave8 + 4 * i;
        return tr ? 8 * (id & 3) + (lane >> 3) : 8 * ((lane & 3) ^ ((lane >> 4) & 3));
    }
    __device__ __forceinline__ int row_of(bool tr, int i) const {
        const int id = wave8 + 4 * i;
        return tr ? (id >> 2) * 64 + 8 * ((lane & 7) ^ (((lane >> 4) & 1) << 2)) : 16 * id + (lane >> 2);
    }
    __device__ __forceinline__ void init(unsigned char* s, int64_t a_ld, int64_t b_ld) {
        smem = s;
        const int tid = (int)threadIdx.x;
        lane = tid & 63;
        wave8 = __builtin_amdgcn_readfirstlane(tid >> 6);
        grp = wave8 >> 1;
        wave = wave8 & 1;
        const int l31 = lane & 31, h = lane >> 5;
#pragma unroll
        for (int i = 0; i < NA; ++i) va[i] = ATR ? (unsigned)(k_of(ATR, i) * a_ld + row_of(ATR, i)) * 2u : (unsigned)(row_of(ATR, i) * a_ld + k_of(ATR, i)) * 2u;
#pragma unroll
        for (int i = 0; i < NB; ++i) vb[i] = BTR ? (unsigned)(k_of(BTR, i) * b_ld + row_of(BTR, i)) * 2u : (unsigned)(row_of(BTR, i) * b_ld + k_of(BTR, i)) * 2u;
        astep = ATR ? LBK * a_ld : LBK;
        bstep = BTR ? LBK * b_ld : LBK;
        const int trl = (8 * h + ((lane & 15) >> 2)) * 128 + (((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ (((lane >> 3) & 1) << 2)) << 4) + (lane & 1) * 8;
        const int nrl = l31 * 64 + ((h ^ ((l31 >> 2) & 3)) << 4);
        const int lds0 = (int)(unsigned)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
        aoff = lds0 + (ATR ? trl + ((grp * MT) >> 1) * 4096 : nrl + grp * MT * 2048);
        boff = lds0 + ABYTES + (BTR ? trl + ((wave * NT) >> 1) * 4096 : nrl + wave * NT * 2048);
        fslot = 0;
    }
    __device__ __forceinline__ void open(const uint16_t* a, int a_rows, const uint16_t* b, int b_rows, int K, const uint32_t* k_mask = nullptr,
                                         const uint32_t* b_mask = nullptr) {
#pragma unroll
        for (int i = 0; i < NA; ++i) ka[i] = KM ? (row_of(ATR, i) < a_rows ? 1 << k_of(ATR, i) : 0) : row_of(ATR, i) < a_rows ? k_of(ATR, i) : 0x40000000;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            bool ok = row_of(BTR, i) < b_rows;
            if (!BTR && b_mask) {  // (a piece is 16 rows: half a word)
                const int id = wave8 + 4 * i;
                ok = ok && ((as_mask(b_mask)[id >> 1] >> ((id & 1) * 16 + (lane >> 2))) & 1);
            }
            kb[i] = ok ? k_of(BTR, i) : 0x40000000;
        }
        ap = a;
        bp = b;
        krem = K;
        if (KM) {
            km = as_mask(k_mask);
            w[0] = km[0];
            w[1] = km[1];
            w[2] = km[2];
            km += 3;
        }
    }
    // KM: ka is the bit of the lane's k, and the stage's word says which k there are
    __device__ __forceinline__ uint32_t a_word() const { return krem >= LBK ? w[0] : krem > 0 ? w[0] & ((1u << krem) - 1) : 0u; }
    __device__ __forceinline__ bool a_ok(int i, uint32_t word) const { return KM ? (ka[i] & (int)word) != 0 : ka[i] < krem; }
    __device__ __forceinline__ uint32_t read_word() { return KM ? *km++ : 0u; }  // (the masks are longer than their numbers by what is read ahead)
    __device__ __forceinline__ void push_word(uint32_t word) {
        w[0] = w[1];
        w[1] = w[2];
        w[2] = word;
    }
    __device__ __forceinline__ void fetch_a(int i) {
        const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)ap, 0, LCAP, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(smem + fslot + wave8 * 1024 + i * 4096), 16,
                                                 (int)(a_ok(i, a_word()) ? va[i] : LSENT), 0, 0, 0);
    }
    __device__ __forceinline__ void fetch_b(int i) {
        const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void*)bp, 0, LCAP, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void*)(smem + fslot + ABYTES + wave8 * 1024 + i * 4096), 16,
                                                 (int)(kb[i] < krem ? vb[i] : LSENT), 0, 0, 0);
    }
    __device__ __forceinline__ void fetched(uint32_t word) {
        ap += astep;
        bp += bstep;
        krem -= LBK;
        if (KM) push_word(word);
        fslot = fslot + STAGE == RING * STAGE ? 0 : fslot + STAGE;
    }
    template <class Next>
    __device__ __forceinline__ void prime(Next&&) {
#pragma unroll
        for (int f = 0; f < RING - 1; ++f) {
#pragma unroll
            for (int i = 0; i < NA; ++i) fetch_a(i);
#pragma unroll
            for (int i = 0; i < NB; ++i) fetch_b(i);
            fetched(read_word());
        }
    }
    __device__ __forceinline__ void start() {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 2) * NPW) : "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    // tile t (32 rows) of the wave's, half kk; asm, so that the compiler waits for no DMA in front of it: the registers become values behind a wait
    template <bool TR>
    __device__ __forceinline__ void read(u32x4& r, u32x2& lo, u32x2& hi, int base, int t, int kk) const {
        if (TR) {
            const int o = (base ^ ((t & 1) << 6)) + (t >> 1) * 4096 + kk * 2048;
            asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(lo) : "v"(o));
            asm volatile("ds_read_b64_tr_b16 %0, %1 offset:512" : "=v"(hi) : "v"(o));
        } else {
            const int o = (base ^ (kk << 5)) + t * 2048;
            asm volatile("ds_read_b128 %0, %1" : "=v"(r) : "v"(o));
        }
    }
    template <bool TR>
    static __device__ __forceinline__ void value(u32x4& r, u32x2& lo, u32x2& hi) {
        if (TR) {
            asm volatile("" : "+v"(lo), "+v"(hi));
            r = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else asm volatile("" : "+v"(r));
    }
    template <class Next>
    __device__ __forceinline__ void run(int steps, f32x16 (&acc)[MT][NT], Next&&) {
        u32x4 a[2][MT], b[2][NT];
        u32x2 al[2][MT], ah[2][MT], bl[2][NT], bh[2][NT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
        int so = 0;
#pragma unroll
        for (int i = 0; i < NT; ++i) read<BTR>(b[0][i], bl[0][i], bh[0][i], boff, i, 0);
#pragma unroll
        for (int i = 0; i < MT; ++i) read<ATR>(a[0][i], al[0][i], ah[0][i], aoff, i, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < NT; ++i) value<BTR>(b[0][i], bl[0][i], bh[0][i]);
#pragma unroll
        for (int i = 0; i < MT; ++i) value<ATR>(a[0][i], al[0][i], ah[0][i]);
        for (int st = 0; st < steps; ++st) {
            const int ab = aoff + so, bb = boff + so;
            so = so + STAGE == RING * STAGE ? 0 : so + STAGE;
            const int an = aoff + so, bn = boff + so;
            if (KM) asm volatile("" : "+s"(w[0]), "+s"(w[1]), "+s"(w[2]));
            const uint32_t word = read_word();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < NT; ++i) read<BTR>(b[1][i], bl[1][i], bh[1][i], bb, i, 1);
#pragma unroll
            for (int i = 0; i < MT; ++i) read<ATR>(a[1][i], al[1][i], ah[1][i], ab, i, 1);
            __builtin_amdgcn_sched_barrier(0);
            // multiply half 0; fetch stage st + RING - 1, into the slot whose last reads ended before the barrier of step st - 1
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                fetch_a(i);
                if (i < NB) fetch_b(i);
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = lmfma<DT>(a[0][i], b[0][j], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            fetched(word);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * NPW) : "memory");  // stage st + 1, and this stage's last fragments
#pragma unroll
            for (int i = 0; i < NT; ++i) value<BTR>(b[1][i], bl[1][i], bh[1][i]);
#pragma unroll
            for (int i = 0; i < MT; ++i) value<ATR>(a[1][i], al[1][i], ah[1][i]);
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            // multiply half 1; read half 0 of the next stage
#pragma unroll
            for (int i = 0; i < NT; ++i) read<BTR>(b[0][i], bl[0][i], bh[0][i], bn, i, 0);
#pragma unroll
            for (int i = 0; i < MT; ++i) read<ATR>(a[0][i], al[0][i], ah[0][i], an, i, 0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = lmfma<DT>(a[1][i], b[1][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int i = 0; i < NT; ++i) value<BTR>(b[0][i], bl[0][i], bh[0][i]);
#pragma unroll
            for (int i = 0; i < MT; ++i) value<ATR>(a[0][i], al[0][i], ah[0][i]);
        }
        drain();
    }
    __device__ __forceinline__ unsigned char* free_slot() const { return smem; }
    __device__ __forceinline__ void settle() {}
    __device__ __forceinline__ void sync() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    __device__ __forceinline__ void drain() {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
};
constexpr int QRING = 4;
template <int DT, int MT, int NT, bool ATR, bool BTR, bool WALK, bool KM>
using Product = std::conditional_t<MT == 4, Pipe<DT, MT, NT, ATR, BTR, WALK, KM>, Quad<DT, MT, NT, ATR, BTR, QRING, KM>>;
template <int MT> constexpr int kLinThreads = MT == 4 ? 512 : 256;
template <int MT, int NT> constexpr int kLinCols = MT == 4 ? NT * 128 : NT * 64;  // B rows of a tile (A rows: MT * 64)

// ---- first product: logits of a tile of classes x rows ------------------------------------------------------------------------------------------
struct LogitArgs {
    const uint16_t* x;
    const uint16_t* w;
    int64_t x_ld, w_ld;
    const float* off;     // [V] class offsets, or null (class_offset)
    float c, coff;        // z / tau in units of log2: acc * c + off * coff
    int N, V, d;          // V, w, off: of the piece in the backward
    int ntv, ntr;         // tiles
    const void* label;    // [N] int64 / int32 (cross entropy) or null
    int label64, v_first; // first class of the piece
    // forward
    float* part;          // [2][nvb][N]: maximum and sum per 32 MT classes
    float* zlab;          // [N] logit of the label (log2 units)
    // backward
    const float* lse2;    // [N] (+inf: the row takes no part)
    const float* coef;    // [N]
    const uint32_t* live; // small tile: bit per row, takes part (the others' features are not read: 0 * inf and NaN stay out)
    uint16_t* dz;         // [rows][dz_ld]
    int64_t dz_ld;
    int dz_rows;          // rows to be written (N rounded up to 32)
    const int32_t* idx;   // small tile only: the teacher's slots, or null
    const float* saved;
    int k;
};

__device__ __forceinline__ int64_t load_label(const void* p, int is64, int r) {
    return is64 ? reinterpret_cast<const int64_t*>(p)[r] : (int64_t)reinterpret_cast<const int32_t*>(p)[r];
}

// dz at the class that slot j of row r names: coef * (p - q)
struct TeacherDz {
    float z2, q, l2, g;
    __device__ __forceinline__ void load(const float* saved, const float* lse2, const float* coef, int k, int r, int j) {
        const float* sv = saved + (int64_t)r * (1 + 2 * k);
        z2 = sv[1 + j];
        q = sv[1 + k + j];
        l2 = lse2[r];
        g = coef[r];
    }
    template <int DT>
    __device__ __forceinline__ void store(uint16_t* at) const {
        if (q == -1.f || l2 == INFINITY || z2 == -INFINITY) return;  // another slot's, or a row without a part, or a left-out class (no gradient)
        *at = Elem<DT>::from_f32((__builtin_amdgcn_exp2f(z2 - l2) - q) * g);
    }
};

// 32 C columns x (HT*32) C rows of 16-bit values through `stg` (wave-private, HT * 2 KiB) as whole rows of the destination: pk[i][q] = the lane's rows
// 32 i + 8 q + 4 h .. +3 of column l31
template <int HT>
__device__ __forceinline__ void store_rows16(unsigned char* stg, const uint2 (&pk)[HT][4], int lane, uint16_t* dst, int64_t ld, int nrows, int ncols) {
    constexpr int RS = HT * 64, CH = HT * 4;  // 16-byte chunk c of row r is kept at c ^ swz(r)
    auto swz = [](int r) { return CH == 8 ? r & 7 : (r >> 1) & 3; };
    const int l31 = lane & 31, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < HT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) *reinterpret_cast<uint2*>(stg + l31 * RS + (((i * 4 + q) ^ swz(l31)) << 4) + h * 8) = pk[i][q];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    u32x4 v[32 * CH / 64];
#pragma unroll
    for (int it = 0; it < 32 * CH / 64; ++it) {
        const int id = it * 64 + lane, row = id / CH, ch = id % CH;
        v[it] = *reinterpret_cast<const u32x4*>(stg + row * RS + ((ch ^ swz(row)) << 4));
    }
#pragma unroll
    for (int it = 0; it < 32 * CH / 64; ++it) {
        const int id = it * 64 + lane, row = id / CH, ch = id % CH;
        if (row < nrows && ch * 8 < ncols) *reinterpret_cast<u32x4*>(dst + row * ld + ch * 8) = v[it];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
// column tile j of the accumulators (TIMES: times f), in halves of MT / 2 row tiles
template <int DT, bool TIMES, int MT, int NT>
__device__ __forceinline__ void store_scaled(unsigned char* stg, const f32x16 (&acc)[MT][NT], int j, float f, int lane, uint16_t* dst, int64_t ld, int nrows, int ncols) {
    constexpr int HT = MT / 2;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint2 pk[HT][4];
#pragma unroll
        for (int i = 0; i < HT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x16& c = acc[half * HT + i][j];
                pk[i][q].x = TIMES ? lpack2<DT>(c[4 * q] * f, c[4 * q + 1] * f) : lpack2<DT>(c[4 * q], c[4 * q + 1]);
                pk[i][q].y = TIMES ? lpack2<DT>(c[4 * q + 2] * f, c[4 * q + 3] * f) : lpack2<DT>(c[4 * q + 2], c[4 * q + 3]);
            }
        store_rows16<HT>(stg, pk, lane, dst + half * HT * 32, ld, nrows, ncols - half * HT * 32);
    }
}

// The large tile's workgroups are persistent, one a CU: each walks its tiles, the next tile's first stages in flight under the epilogue (4096 x 65536 x 640
// bf16: 363 -> 327 us forward). A launch of the small tile has one tile a workgroup and skips that bookkeeping (96 x 365 x 320: 8.4 us with it, 6.3 without).
// Panels of 8 row tiles; an XCD's workgroups take neighbouring tiles: together 8 row tiles x 4 class tiles at a time, whose operands its L2 hands out.
template <int DT, int MT, int NT, bool BWD>
__global__ __launch_bounds__(kLinThreads<MT>, 2) void class_logits_kernel(const LogitArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int BM = MT * 64, BN = kLinCols<MT, NT>, GR = 8;
    constexpr bool WALK = MT == 4;
    const int ntiles = a.ntv * a.ntr;
    int L, end, per = 1;
    if (WALK) {
        const int nwg = (int)gridDim.x, xcd = (int)blockIdx.x & 7;
        per = (nwg - xcd + 7) >> 3;  // workgroups of this XCD
        const int q8 = ntiles >> 3, r8 = ntiles & 7;
        const int first = xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8;
        end = first + q8 + (xcd < r8 ? 1 : 0);
        L = first + ((int)blockIdx.x >> 3);
        if (L >= end) return;
    } else {
        L = xcd_order((int)blockIdx.x, (int)gridDim.x);
        end = L + 1;
    }
    int v0, r0;                      // of the tile that is multiplied
    auto place = [&](int t, int& v, int& r) {
        const int panel = t / (GR * a.ntv), pr0 = panel * GR, pw = min(GR, a.ntr - pr0), in = t - panel * GR * a.ntv;
        v = in / pw * BM;
        r = (pr0 + in % pw) * BN;
    };
    place(L, v0, r0);
    Product<DT, MT, NT, false, false, WALK, false> p;
    p.init(smem, a.w_ld, a.x_ld);
    int F = L;                       // the tile that is fetched
    auto open = [&]() {
        int v = v0, r = r0;
        const bool more = F < end;
        if (WALK && more && F != L) place(F, v, r);
        const uint16_t *w = a.w + (int64_t)v * a.w_ld, *x = a.x + (int64_t)r * a.x_ld;
        if constexpr (WALK) p.open(w, more ? a.V - v : 0, x, more ? a.N - r : 0, a.d);
        else p.open(w, a.V - v, x, a.N - r, a.d, nullptr, BWD ? a.live + (r >> 5) : nullptr);
        F += per;
    };
    // offsets of a tile's classes in log2 units, -inf for those left out or behind the last, and which of the writing waves met one. Walking: two tables behind
    // the ring, the next tile's written a tile ahead; else one, in the ring when that has ended
    constexpr int TABLE = BM + 4, STAGE = Product<DT, MT, NT, false, false, WALK, false>::STAGE;
    float* table = reinterpret_cast<float*>(smem + LRING * STAGE);
    const bool writer = a.off && (int)threadIdx.x < BM;
    auto offset = [&](int t) {
        int v = v0, r;
        if (WALK && t != L) place(t, v, r);
        v += (int)threadIdx.x;
        return v < a.V ? class_offset(a.off[v], a.coff) : -INFINITY;
    };
    auto note = [&](float* dst, float o) {
        dst[threadIdx.x] = o;
        const bool out = __ballot(o == -INFINITY) != 0;
        if (p.lane == 0) reinterpret_cast<int*>(dst + BM)[p.wave8] = out;
    };
    int turn = 0;
    open();
    const float o_first = writer ? offset(L) : 0.f;
    p.prime(open);
    if (WALK && writer) note(table, o_first);
    p.start();
    const int lane = p.lane, l31 = lane & 31, h = lane >> 5, grp = p.grp, wave = p.wave, steps = (a.d + LBK - 1) / LBK;
    for (;;) {
        f32x16 acc[MT][NT];
        p.run(steps, acc, open);
        if (!WALK && a.off) {
            table = reinterpret_cast<float*>(smem + STAGE);  // (results are staged in free_slot())
            if (writer) note(table, o_first);
            p.sync();
        }
        const int vw = v0 + grp * MT * 32;               // the wave's first class
        unsigned char* stg = p.free_slot() + p.wave8 * (MT * 1024);
        const float* const offw = table + turn * TABLE + grp * MT * 32;
        const int* const outs = reinterpret_cast<const int*>(table + turn * TABLE + BM);
        turn ^= 1;
        if (WALK && writer && L + per < end) note(table + turn * TABLE, offset(L + per));
        // classes with an offset, or behind the last one: the logits themselves take the accumulators' place (the product's sign matters to the maximum)
        float c = a.c;
        if (a.off || v0 + BM > a.V || (!BWD && c <= 0.f)) {
            bool out = v0 + BM > a.V;
            if (a.off)
#pragma unroll
                for (int i = 0; i < BM / 64; ++i) out = out || outs[i];
            f32x4 o[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) o[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (a.off) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) o[i][q] = *reinterpret_cast<const f32x4*>(offw + i * 32 + q * 8 + h * 4);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < NT; ++j) acc[i][j][4 * q + e] = fmaf(acc[i][j][4 * q + e], c, o[i][q][e]);
            if (out) {  // -inf whatever the weights hold: 0 * inf and NaN stay out
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool gone = o[i][q][e] == -INFINITY || vw + i * 32 + q * 8 + h * 4 + e >= a.V;
#pragma unroll
                            for (int j = 0; j < NT; ++j) acc[i][j][4 * q + e] = gone ? -INFINITY : acc[i][j][4 * q + e];
                        }
            }
            c = 1.f;
        }
        if (!BWD) {
            float mu[NT], s[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float m = -INFINITY;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[i][j][e]);
                m = fmaxf(m, __shfl_xor(m, 32)) * c;
                mu[j] = __builtin_isinf(m) ? 0.f : m;  // nothing left, or an infinite logit: exp2 of the values themselves
                s[j] = 0.f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[j] += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -mu[j]));
                s[j] += __shfl_xor(s[j], 32);
            }
            float zl[NT];
            bool mine[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int r = r0 + (wave * NT + j) * 32 + l31;
                const int64_t at = a.label && r < a.N ? load_label(a.label, a.label64, r) - vw : -1;
                mine[j] = at >= 0 && at < MT * 32 && (((int)at >> 2) & 1) == h;
                zl[j] = 0.f;
                if (__ballot(mine[j])) {
                    const int slot = (((int)at >> 3) << 2) | ((int)at & 3);  // (i, q, e) of the lane that holds it
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) zl[j] = slot == i * 16 + e ? acc[i][j][e] : zl[j];
                }
            }
            p.settle();
            const int64_t vb = (int64_t)(vw / (MT * 32)), nvb = (int64_t)a.ntv * 2;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int r = r0 + (wave * NT + j) * 32 + l31;
                if (mine[j]) a.zlab[r] = zl[j] * c;
                if (h == 0 && r < a.N) {
                    a.part[vb * a.N + r] = mu[j];
                    a.part[(nvb + vb) * a.N + r] = s[j];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int r = r0 + (wave * NT + j) * 32 + l31;
                const bool live = r < a.N;
                const float l2 = live ? a.lse2[r] : INFINITY, g = live ? a.coef[r] : 0.f, mag = fabsf(g);
                const int64_t at = a.label && live ? load_label(a.label, a.label64, r) - a.v_first - vw : -1;
                const float l2g = l2 - __builtin_amdgcn_logf(mag);  // |g| p = exp2(t - lse + log2 |g|): nothing for g = 0
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], c, -l2g));
                bool mine = at >= 0 && at < MT * 32 && vw + at < a.V && (((int)at >> 2) & 1) == h;
                if (a.off && mine) mine = offw[(int)at] != -INFINITY;  // (a left-out class gets no gradient)
                if (__ballot(mine)) {
                    const int slot = (((int)at >> 3) << 2) | ((int)at & 3);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][j][e] -= mine && slot == i * 16 + e ? mag : 0.f;
                }
                if (__ballot(g < 0.f)) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][j][e] = g < 0.f ? -acc[i][j][e] : acc[i][j][e];
                }
            }
            p.settle();
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int rr = r0 + (wave * NT + j) * 32;
                store_scaled<DT, false>(stg, acc, j, 1.f, lane, a.dz + (int64_t)rr * a.dz_ld + vw, a.dz_ld, a.dz_rows - rr, MT * 32);
            }
        }
        if (!WALK && BWD && a.idx) {
            __syncthreads();  // the tile is written: the entries that the teacher names may follow
            const int rows = min(BN, a.N - r0), V = min(BM, a.V - v0);
            constexpr int U = 8;  // slots of a thread in flight
            const int n = rows * a.k;
            for (int i0 = (int)threadIdx.x; i0 < n; i0 += U * kLinThreads<MT>) {
                int v[U], r[U];
                TeacherDz t[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * kLinThreads<MT>;
                    v[u] = -1;
                    if (i >= n) continue;
                    r[u] = r0 + i / a.k;
                    v[u] = a.idx[(int64_t)r0 * a.k + i] - a.v_first - v0;
                    t[u].load(a.saved, a.lse2, a.coef, a.k, r[u], i % a.k);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if ((unsigned)v[u] < (unsigned)V) t[u].template store<DT>(a.dz + r[u] * a.dz_ld + v0 + v[u]);
            }
        }
        L += per;
        if (!WALK || L >= end) break;
        p.sync();
        place(L, v0, r0);
    }
    p.drain();
}

// ---- second product of the backward: a piece's dw tiles and dx tiles in one launch -----------------------------------------------------------------
struct GradArgs {
    const uint16_t* x;    // [N][x_ld]; large tile: with zeros in the rows that take no part
    const uint16_t* w;    // [Vp][w_ld], first class of the piece
    const uint16_t* dz;   // [rows32][dz_ld]
    const uint32_t *live, *kept;  // bit per row, takes part (small tile); per class of the piece, not left out. The others are not read: 0 * inf and NaN stay out
    int64_t x_ld, w_ld, dz_ld;
    int N, rows32, d, Vp; // Vp: classes of the piece
    int vk;               // columns of dz that hold numbers (Vp rounded up to the tile)
    int ntd, ndw, ndx;    // tiles along d; dw tiles, dx tiles
    int dx_first;
    int ntr, kper;        // dx: row tiles, classes per slice of the piece (a multiple of 32)
    int wsplits, rper;    // dw: slices of the rows, rows per slice (a multiple of 32)
    uint16_t* dw;         // [Vp][dw_ld]
    int64_t dw_ld;
    uint16_t* dx;         // one piece, one slice: dx itself; else null and
    int64_t dx_ld;
    float* slab;          // dx [slices][N][d], and
    int add;              // whether it holds earlier pieces
    float* wslab;         // more than one slice of the rows: [slices][Vp][d]
    const float* outscale;
};

// (The large tile has 256 registers a lane, and its two forms spill 2 and 5 of them where a tile is added to its slab.)
// KEPT: classes can be left out, whose weights are not read (1021 x 32003 x 512: 2 us in the loop, a copy of w with zeros there 10; 494 x 63581 x 984 50)
template <int DT, int MT, int NT, bool KEPT>
__global__ __launch_bounds__(kLinThreads<MT>, 2) void class_grads_kernel(const GradArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int BM = MT * 64, BN = kLinCols<MT, NT>;
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int wave8 = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int WN = MT == 4 ? 4 : 2;  // waves along the tile's columns
    const int grp = wave8 / WN, wave = wave8 % WN, l31 = lane & 31, h = lane >> 5;
    // every XCD gets its even share of the dw tiles and of the dx tiles (neighbouring ones), the longer kind first
    int L;
    bool is_dw;
    {
        const int xcd = (int)blockIdx.x & 7, j = (int)blockIdx.x >> 3, n = (int)gridDim.x;
        auto start = [&](int count) { return (count >> 3) * xcd + min(xcd, count & 7); };  // of this XCD's share of `count`
        const int dw0 = start(a.ndw), dwn = (a.ndw >> 3) + (xcd < (a.ndw & 7) ? 1 : 0), dx0 = start(n) - dw0, dxn = (n >> 3) + (xcd < (n & 7) ? 1 : 0) - dwn;
        is_dw = a.dx_first ? j >= dxn : j < dwn;
        L = is_dw ? dw0 + (a.dx_first ? j - dxn : j) : dx0 + (a.dx_first ? j : j - dwn);
    }
    unsigned char* stg = smem + wave8 * (MT * 1024);
    f32x16 acc[MT][NT];
    // column tile j of the accumulators onto rows of a slab
    auto onto = [&](float* slab, int j, int row0, int rows, int f0, bool add) {
        const int r = row0 + (wave * NT + j) * 32 + l31;
        if (r >= rows) return;
        f32x4 *p = reinterpret_cast<f32x4*>(slab + (int64_t)r * a.d), old[MT][4];
        const int c0 = f0 + grp * MT * 32 + h * 4;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                old[i][q] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (add && c0 + i * 32 + q * 8 < a.d) old[i][q] = p[(c0 + i * 32 + q * 8) >> 2];
            }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c0 + i * 32 + q * 8 < a.d)
                    p[(c0 + i * 32 + q * 8) >> 2] = old[i][q] + f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    };
    if (is_dw) {  // dw[v][f] = sum over the slice's rows of dz[r][v] x[r][f]
        const int nvt = a.ndw / (a.ntd * a.wsplits), f0 = (L % a.ntd) * BM, v0 = (L / a.ntd % nvt) * BN, s = L / a.ntd / nvt;
        const int k0 = min(s * a.rper, a.N), k = min(a.rper, a.N - k0);
        Product<DT, MT, NT, true, true, false, MT == 2> p;
        auto none = []() {};
        p.init(smem, a.x_ld, a.dz_ld);
        const uint16_t *x = a.x + (int64_t)k0 * a.x_ld + f0, *dz = a.dz + (int64_t)k0 * a.dz_ld + v0;
        if constexpr (MT == 4) p.open(x, a.d - f0, dz, a.vk - v0, k);
        else p.open(x, a.d - f0, dz, a.vk - v0, k, a.live + (k0 >> 5));
        p.prime(none);
        p.start();
        p.run((k + LBK - 1) / LBK, acc, none);
        p.drain();
        if (a.wsplits > 1) {
#pragma unroll
            for (int j = 0; j < NT; ++j) onto(a.wslab + (int64_t)s * a.Vp * a.d, j, v0, a.Vp, f0, false);
            return;
        }
        const float os = *a.outscale;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int v = v0 + (wave * NT + j) * 32, f = f0 + grp * MT * 32;
            store_scaled<DT, true>(stg, acc, j, os, lane, a.dw + (int64_t)v * a.dw_ld + f, a.dw_ld, a.Vp - v, a.d - f);
        }
        return;
    }
    // dx[r][f] += sum over the slice's classes of dz[r][v] w[v][f]
    const int f0 = (L % a.ntd) * BM, r0 = (L / a.ntd % a.ntr) * BN, s = L / a.ntd / a.ntr;
    const int k0 = min(s * a.kper, a.Vp), k = min(a.kper, a.Vp - k0);
    {
        Product<DT, MT, NT, true, false, false, KEPT> p;
        auto none = []() {};
        p.init(smem, a.w_ld, a.dz_ld);
        const uint16_t *w = a.w + (int64_t)k0 * a.w_ld + f0, *dz = a.dz + (int64_t)r0 * a.dz_ld + k0;
        if constexpr (!KEPT) p.open(w, a.d - f0, dz, a.rows32 - r0, k);
        else p.open(w, a.d - f0, dz, a.rows32 - r0, k, a.kept + (k0 >> 5));
        p.prime(none);
        p.start();
        p.run((k + LBK - 1) / LBK, acc, none);
        p.drain();
    }
    if (a.dx) {
        const float os = *a.outscale;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = r0 + (wave * NT + j) * 32, f = f0 + grp * MT * 32;
            store_scaled<DT, true>(stg, acc, j, os, lane, a.dx + (int64_t)r * a.dx_ld + f, a.dx_ld, a.N - r, a.d - f);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) onto(a.slab + (int64_t)s * a.N * a.d, j, r0, a.N, f0, a.add);
}

// ---- small launches ----------------------------------------------------------------------------------------------------------------------------------
// rows' (maximum, sum) pairs -> lse: C rows a workgroup (a power of two), 1024 / C threads a row that take every (1024 / C)th pair, joined in a tree of
// fixed order
// a sum of 0 has no maximum; one of inf, whose maximum is written as 0, stays inf beside any other (and does not become inf * 0), NaN stays NaN
__device__ __forceinline__ void lse_join(float& m, float& s, float m2, float s2) {
    if (s2 == 0.f) return;
    if (s == 0.f) {
        m = m2;
        s = s2;
        return;
    }
    const float mn = fmaxf(m, m2);
    s = (s == INFINITY ? s : s * __builtin_amdgcn_exp2f(m - mn)) + (s2 == INFINITY ? s2 : s2 * __builtin_amdgcn_exp2f(m2 - mn));
    m = mn;
}
__global__ __launch_bounds__(1024) void class_lse_kernel(const float* part, int nvb, int N, int V, int C, const void* label, int label64, const float* zlab, float* loss,
                                                         float* lse) {
    __shared__ float sm[1024], ss[1024];
    const int t = (int)threadIdx.x, c = t & (C - 1), G = 1024 / C, g = t / C;
    const int r = (int)blockIdx.x * C + c;
    float m = 0.f, s = 0.f;
    if (r < N) {
        const float *pm = part + r, *ps = part + (int64_t)nvb * N + r;
        for (int b = g; b < nvb; b += 4 * G) {
            float m4[4], s4[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool in = b + u * G < nvb;
                m4[u] = in ? pm[(int64_t)(b + u * G) * N] : 0.f;
                s4[u] = in ? ps[(int64_t)(b + u * G) * N] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) lse_join(m, s, m4[u], s4[u]);
        }
    }
    sm[t] = m;
    ss[t] = s;
    for (int o = G >> 1; o; o >>= 1) {
        __syncthreads();
        if (g < o) {
            lse_join(m, s, sm[t + o * C], ss[t + o * C]);
            sm[t] = m;
            ss[t] = s;
        }
    }
    if (g || r >= N) return;
    const float l2 = s == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(s);  // (v_log_f32: base 2)
    lse[r] = l2 * kLn2;
    if (loss) {
        const int64_t lab = load_label(label, label64, r);
        loss[r] = lab >= 0 && lab < V && s != 0.f ? (l2 - zlab[r]) * kLn2 : 0.f;
    }
}

// What the backward needs of every row -- lse, coefficient, whether it takes part -- and which classes are not left out; and, for the large tile, x with
// zeros in the rows that take no part (0 * inf and NaN stay out).
// A row's coefficient is g_r times what brings the largest |g| of the rows that take part to 1.984375 (fp16: times 2^12): the entries of dz that matter
// most, g (p - 1) at the labels of rows with the largest weight (of all rows, under a mean), then lie at the top of a binade, where rounding to 16 bits
// costs half of what it does at its bottom; and dz stays inside fp16's range. Every workgroup finds the maximum for itself (N up to 32768: 16 bytes a row
// out of the L2), or is given it.
struct PrepArgs {
    const float* drow;
    int drow_stride;
    const void* label;
    int label64;
    const float* lse;
    int64_t lse_stride;
    int N, V;
    float gain, spread;
    const float* gmax;          // null: find it
    const float* off;           // [V] or null
    float coff;                 // as LogitArgs
    float *lse2, *coef, *outscale;
    uint32_t *live, *kept;
    const uint16_t* x;          // null: no copy
    int64_t x_ld;
    int d8;
    u32x4* xo;
};
__device__ __forceinline__ bool prep_live(const PrepArgs& a, int64_t r) {
    const float l = a.lse[r * a.lse_stride];
    if (!a.label) return l != INFINITY;  // (the teacher's mark)
    if (l == -INFINITY) return false;
    const int64_t lab = load_label(a.label, a.label64, r);
    return lab >= 0 && lab < a.V;
}
__device__ __forceinline__ float prep_max(const PrepArgs& a) {  // 1024 threads
    __shared__ float red[16];
    const int t = (int)threadIdx.x;
    float m = 0.f;
    for (int r = t; r < a.N; r += 1024) {
        const float g = a.drow ? fabsf(a.drow[(int64_t)r * a.drow_stride]) : 1.f;
        if (g <= 3.4e38f && g > m && prep_live(a, r)) m = g;
    }
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((t & 63) == 0) red[t >> 6] = m;
    __syncthreads();
    m = red[0];
    for (int i = 1; i < 16; ++i) m = fmaxf(m, red[i]);
    return m;
}
__global__ __launch_bounds__(1024) void class_max_kernel(const PrepArgs a, float* out) {
    const float m = prep_max(a);
    if (threadIdx.x == 0) *out = m;
}
__global__ __launch_bounds__(1024) void class_prep_kernel(const PrepArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 1024 + threadIdx.x, nt = (int64_t)gridDim.x * 1024;
    float m = a.gmax ? *a.gmax : prep_max(a);
    m = m > 0.f ? fminf(fmaxf(m, 1e-30f), 1e37f) : 1.f;
    const float down = 1.984375f * a.spread / m;
    for (int64_t r = t; r - (t & 63) < a.N; r += nt) {  // (whole waves: a wave writes 64 bits)
        const bool on = r < a.N && prep_live(a, r);
        const uint64_t bits = __ballot(on);
        if ((t & 63) == 0) *reinterpret_cast<uint64_t*>(a.live + (r >> 5)) = bits;
        if (r >= a.N) continue;
        const float g = a.drow ? a.drow[r * a.drow_stride] : 1.f;
        const float l = a.lse[r * a.lse_stride] * kLog2e;
        a.lse2[r] = !on ? INFINITY : l == INFINITY ? NAN : l;  // +inf marks a row without a part; an infinite logit gives NaN gradients
        a.coef[r] = on ? g * down : 0.f;
    }
    for (int64_t v = t; v - (t & 63) < a.V; v += nt) {
        const uint64_t bits = __ballot(v < a.V && (!a.off || class_offset(a.off[v], a.coff) != -INFINITY));
        if ((t & 63) == 0) *reinterpret_cast<uint64_t*>(a.kept + (v >> 5)) = bits;
    }
    if (t == 0) *a.outscale = a.gain * m / (1.984375f * a.spread);
    if (a.x)
        for (int64_t i = t; i < (int64_t)a.N * a.d8; i += nt) {
            const int64_t r = i / a.d8, c = i - r * a.d8;
            a.xo[i] = prep_live(a, r) ? *reinterpret_cast<const u32x4*>(a.x + r * a.x_ld + c * 8) : u32x4{0, 0, 0, 0};
        }
}
struct SumArgs {
    const float* slab[2];
    uint16_t* out[2];
    int64_t ld[2];
    int rows[2], slices[2];
    int d;
    const float* outscale;
};
template <int DT>
__global__ __launch_bounds__(256) void class_sum_kernel(const SumArgs a) {
    const int w = (int)blockIdx.y, d4 = a.d >> 2, slices = a.slices[w];
    const int64_t n = (int64_t)a.rows[w] * d4, ld = a.ld[w];
    const f32x4* slab = reinterpret_cast<const f32x4*>(a.slab[w]);
    uint16_t* out = a.out[w];
    const float os = *a.outscale;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        f32x4 v = slab[i];
        for (int s = 1; s < slices; ++s) v += slab[(int64_t)s * n + i];
        const int64_t r = i / d4;
        uint2 o;
        o.x = lpack2<DT>(v[0] * os, v[1] * os);
        o.y = lpack2<DT>(v[2] * os, v[3] * os);
        *reinterpret_cast<uint2*>(out + r * ld + (i - r * d4) * 4) = o;
    }
}
__global__ __launch_bounds__(256) void class_zero_kernel(uint16_t* p, int64_t rows, int64_t ld, int d) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows * d; i += (int64_t)gridDim.x * 256) p[i / d * ld + i % d] = 0;
}

// ---- backward of few rows ------------------------------------------------------------------------------------------------------------------------------
// At most 128 rows: the class list is what there is to read, so one launch does with one read of it what the tiles above do with two and four launches.
// A workgroup holds x in LDS and walks over blocks of 32 classes, the next block's weights on the way to registers under this one's products:
//   z [classes][rows] = w x^T, K = d shared out to the waves and joined in LDS;  dz, 16-bit, in both orders -- up to 64 rows as two such numbers, the
//   second what the first one's rounding leaves: a row's few large entries average no roundings, and the products wait for memory (from 65 rows on they
//   do not: 128 x 131072 x 320 87 us with one, 110 with two);
//   dw block = dz x, written out;  dx += dz w, in registers until the end: one fp32 slice a workgroup (class_few_sum_kernel adds them in their order).
// A wave owns FT tiles of 32 features in the last two; RT tiles of 32 rows. Bound by memory for long lists, w in and dw out: backward of 1 x 131072 x 960
// 104 us = 4.8 TB/s (by tiles of 128 x 128: 180), 32 x 131072 x 512 68 us (97), 128 x 131072 x 320 90 us (97); of short ones by a chain of waits: 96 x 365 x
// 320 15 + 4 us of kernels (21). Two workgroups a CU where registers and LDS leave room: 16 x 131072 x 400 50 us, with one 59, by tiles 89.
struct FewArgs {
    const uint16_t *x, *w;
    int64_t x_ld, w_ld;
    const float* off;
    float c, coff;
    int N, V, d;
    const void* label;
    int label64;
    const int32_t* idx;   // the teacher's slots (at most kFewSlots * 512), or null
    const float* saved;
    int k;
    const float* lse;
    int64_t lse_stride;
    const float* drow;
    int drow_stride;
    float gain, spread;   // as PrepArgs
    uint16_t* dw;         // or null
    int64_t dw_ld;
    float* slab;          // dx [workgroups][N][d], or null
    float* outscale;
};
constexpr int kFewSlots = 8;
static inline int few_lds(int RT, int N, int d) {  // (x: rows up to the next 16)
    const int S = (d + 31) / 32 * 64 + 16;
    return ((N + 15) / 16 * 16 + 32) * S + 32768 + RT * 32 * 80 + 32 * (RT * 64 + 16) + (RT * 32 * 4 + 64) * 4;
}
__device__ __forceinline__ u32x4 few_row(const unsigned char* p) { return *reinterpret_cast<const u32x4*>(p); }
// features f0 .. +31 as fragment rows, K = lines k0 .. +15 of S bytes
__device__ __forceinline__ u32x4 few_tr(const unsigned char* base, int S, int k0, int f0, int lane) {
    typedef s16x4 __attribute__((address_space(3))) * lds_t;
    const unsigned char* p = base + (k0 + 8 * (lane >> 5) + ((lane & 15) >> 2)) * S + (f0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4) * 2;
    const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p)),
                hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + 4 * S)));
    return u32x4{lo.x, lo.y, hi.x, hi.y};
}
__device__ __forceinline__ void few_sync() {  // LDS only: loads in flight stay in flight
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}
template <int DT, int RT, int FT>
__global__ __launch_bounds__(512, RT * FT <= 2 ? 4 : 2) void class_few_kernel(const FewArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    constexpr int KP = 8 / RT, CS = RT * 64 + 16, WP = FT * 2;
    constexpr bool TWO = RT <= 2;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, h = lane >> 5;
    const int nft = (a.d + 31) >> 5, S = nft * 64 + 16, nch = (a.V + 31) >> 5, step = (int)gridDim.x;
    const int lines = (a.N + 15) & ~15;
    unsigned char *xs = smem, *ws = xs + lines * S, *red = ws + 32 * S, *dzr = red + 32768, *dzc = dzr + RT * 32 * 80, *lor = red, *loc = red + RT * 32 * 80;
    float *l2s = reinterpret_cast<float*>(dzc + 32 * CS), *gs = l2s + RT * 32, *gm = gs + RT * 32, *offs = gm + RT * 32;
    int* labs = reinterpret_cast<int*>(offs + 64);
    int ch = (int)blockIdx.x;
    // a block's weights, the wave's own features of them; offsets (-inf: left out, or behind the last class)
    u32x4 wr[WP];
    float on = 0.f;
    auto fetch = [&](int b) {
#pragma unroll
        for (int i = 0; i < WP; ++i) {
            const int p = lane + 64 * i, v = b * 32 + p / (FT * 4), col = (wave * FT * 4 + p % (FT * 4)) * 8;
            wr[i] = v < a.V && col < a.d ? *reinterpret_cast<const u32x4*>(a.w + v * a.w_ld + col) : u32x4{0, 0, 0, 0};
        }
        if (tid < 32) on = b * 32 + tid >= a.V ? -INFINITY : a.off ? class_offset(a.off[b * 32 + tid], a.coff) : 0.f;
    };
    fetch(ch);
    int sv[kFewSlots];
#pragma unroll
    for (int u = 0; u < kFewSlots; ++u) sv[u] = a.idx && tid + 512 * u < a.N * a.k ? a.idx[tid + 512 * u] : -1;
    // x, zeros in the rows that take no part (known later) and behind the last feature
    u32x4 xv[RT * 4];
    auto load_x = [&](int p) {
#pragma unroll
        for (int i = 0; i < RT * 4; ++i) {
            const int r = wave + 8 * i;
            xv[i] = p * 8 < a.d && r < a.N ? *reinterpret_cast<const u32x4*>(a.x + r * a.x_ld + p * 8) : u32x4{0, 0, 0, 0};
        }
    };
    auto keep = [&](int p) {
        if (p < nft * 4)
#pragma unroll
            for (int i = 0; i < RT * 4; ++i)
                if (wave + 8 * i < lines) *reinterpret_cast<u32x4*>(xs + (wave + 8 * i) * S + p * 16) = l2s[wave + 8 * i] != INFINITY ? xv[i] : u32x4{0, 0, 0, 0};
    };
    load_x(lane);
    if (tid < RT * 32) {  // the rows, as class_prep_kernel has them
        const int r = tid;
        float l = r < a.N ? a.lse[r * a.lse_stride] : 0.f, g = r < a.N ? (a.drow ? a.drow[(int64_t)r * a.drow_stride] : 1.f) : 0.f;
        const int64_t lab = a.label && r < a.N ? load_label(a.label, a.label64, r) : -1;
        const bool live = r < a.N && (a.label ? l != -INFINITY && lab >= 0 && lab < a.V : l != INFINITY);
        l *= kLog2e;
        l2s[r] = !live ? INFINITY : l == INFINITY ? NAN : l;
        gs[r] = live ? g : 0.f;
        gm[r] = live && fabsf(g) <= 3.4e38f ? fabsf(g) : 0.f;
        labs[r] = live ? (int)lab : -1;
    }
    if (tid < 32) offs[tid] = on;
    __syncthreads();
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < (RT + 1) / 2; ++i) m = fmaxf(m, gm[(lane + 64 * i) & (RT * 32 - 1)]);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    m = m > 0.f ? fminf(fmaxf(m, 1e-30f), 1e37f) : 1.f;
    const float down = 1.984375f * a.spread / m, os = a.gain * m / (1.984375f * a.spread);
    if (blockIdx.x == 0 && tid == 0) *a.outscale = os;
    keep(lane);
    for (int p = lane + 64; p < nft * 4; p += 64) {
        load_x(p);
        keep(p);
    }
    __builtin_amdgcn_sched_barrier(0);
    f32x16 acc[RT][FT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < FT; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[t][i][e] = 0.f;
    const int t0 = wave % RT, kp = wave / RT;
    for (int buf = 0; ch < nch; ch += step, buf ^= 32) {
        int ln = (int)threadIdx.x & 63;
        asm volatile("" : "+v"(ln));  // (addresses are computed anew for every block: kept across the loop they cost more registers than there are)
        const int lane = ln, l31 = lane & 31, h = lane >> 5, tid = wave * 64 + lane;
#pragma unroll
        for (int i = 0; i < WP; ++i) {
            const int p = lane + 64 * i, row = p / (FT * 4), at = wave * FT * 4 + p % (FT * 4);
            if (at < nft * 4) *reinterpret_cast<u32x4*>(ws + row * S + at * 16) = offs[buf + row] == -INFINITY ? u32x4{0, 0, 0, 0} : wr[i];
        }
        if (ch + step < nch) fetch(ch + step);
        few_sync();
        f32x16 z;
#pragma unroll
        for (int e = 0; e < 16; ++e) z[e] = 0.f;
        const unsigned char *wz = ws + l31 * S + h * 16, *xz = xs + min(t0 * 32 + l31, lines - 1) * S + h * 16;  // (rows behind the last: any, their dz is 0)
#pragma unroll 4
        for (int s = kp; s < 2 * nft; s += KP) z = lmfma<DT>(few_row(wz + s * 32), few_row(xz + s * 32), z);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(red + (wave * 32 + l31) * 128 + (((2 * q + h) ^ (l31 & 7)) << 4)) = f32x4{z[4 * q], z[4 * q + 1], z[4 * q + 2], z[4 * q + 3]};
        if (tid < 32) offs[(buf ^ 32) + tid] = on;
        few_sync();
        // two classes of RT rows a thread
        const int r31 = tid >> 4, cp = tid & 15;
        const float2 o = *reinterpret_cast<const float2*>(offs + buf + 2 * cp);
        float2 sums[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            sums[t] = float2{0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KP; ++j) {
                const float2 u = *reinterpret_cast<const float2*>(red + ((j * RT + t) * 32 + r31) * 128 + (((cp >> 1) ^ (r31 & 7)) << 4) + (cp & 1) * 8);
                sums[t].x += u.x;
                sums[t].y += u.y;
            }
        }
        if (TWO) few_sync();  // (the rests take the place of the sums)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const float2 s = sums[t];
            const int r = t * 32 + r31, at = labs[r] - ch * 32 - 2 * cp;
            const float l2 = l2s[r], g = gs[r] * down, mag = fabsf(g), l2g = l2 - __builtin_amdgcn_logf(mag);
            float d0 = __builtin_amdgcn_exp2f(fmaf(s.x, a.c, o.x) - l2g), d1 = __builtin_amdgcn_exp2f(fmaf(s.y, a.c, o.y) - l2g);
            d0 -= at == 0 ? mag : 0.f;
            d1 -= at == 1 ? mag : 0.f;
            d0 = o.x == -INFINITY || l2 == INFINITY ? 0.f : g < 0.f ? -d0 : d0;
            d1 = o.y == -INFINITY || l2 == INFINITY ? 0.f : g < 0.f ? -d1 : d1;
            const uint32_t pk = lpack2<DT>(d0, d1);
            *reinterpret_cast<uint32_t*>(dzr + r * 80 + cp * 4) = pk;
            *reinterpret_cast<uint16_t*>(dzc + 2 * cp * CS + r * 2) = (uint16_t)pk;
            *reinterpret_cast<uint16_t*>(dzc + (2 * cp + 1) * CS + r * 2) = (uint16_t)(pk >> 16);
            if (TWO) {
                const uint32_t rest = lpack2<DT>(d0 - Elem<DT>::to_f32((uint16_t)pk), d1 - Elem<DT>::to_f32((uint16_t)(pk >> 16)));
                *reinterpret_cast<uint32_t*>(lor + r * 80 + cp * 4) = rest;
                *reinterpret_cast<uint16_t*>(loc + 2 * cp * CS + r * 2) = (uint16_t)rest;
                *reinterpret_cast<uint16_t*>(loc + (2 * cp + 1) * CS + r * 2) = (uint16_t)(rest >> 16);
            }
        }
        few_sync();
        if (a.idx) {  // the classes that the teacher names
#pragma unroll
            for (int u = 0; u < kFewSlots; ++u) {
                const unsigned v = (unsigned)sv[u] - (unsigned)ch * 32u;
                if (v >= 32u) continue;
                const int i = tid + 512 * u, r = i / a.k, j = i - r * a.k;
                const float z2 = a.saved[(int64_t)r * (1 + 2 * a.k) + 1 + j], q = a.saved[(int64_t)r * (1 + 2 * a.k) + 1 + a.k + j], l2 = l2s[r];
                if (q == -1.f || l2 == INFINITY || z2 == -INFINITY) continue;  // (TeacherDz)
                const float dz = (__builtin_amdgcn_exp2f(z2 - l2) - q) * (gs[r] * down);
                const uint16_t b = Elem<DT>::from_f32(dz);
                *reinterpret_cast<uint16_t*>(dzr + r * 80 + v * 2) = b;
                *reinterpret_cast<uint16_t*>(dzc + v * CS + r * 2) = b;
                if (TWO) {
                    const uint16_t rest = Elem<DT>::from_f32(dz - Elem<DT>::to_f32(b));
                    *reinterpret_cast<uint16_t*>(lor + r * 80 + v * 2) = rest;
                    *reinterpret_cast<uint16_t*>(loc + v * CS + r * 2) = rest;
                }
            }
            few_sync();
        }
#pragma unroll
        for (int i = 0; i < FT; ++i) {
            const int f0 = (wave * FT + i) * 32;
            if (f0 >= a.d) break;
            if (a.slab) {
                const u32x4 w0 = few_tr(ws, S, 0, f0, lane), w1 = few_tr(ws, S, 16, f0, lane);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const int b = (t * 32 + l31) * 80 + h * 16;
                    acc[t][i] = lmfma<DT>(w0, few_row(dzr + b), acc[t][i]);
                    acc[t][i] = lmfma<DT>(w1, few_row(dzr + b + 32), acc[t][i]);
                    if (TWO) {
                        acc[t][i] = lmfma<DT>(w0, few_row(lor + b), acc[t][i]);
                        acc[t][i] = lmfma<DT>(w1, few_row(lor + b + 32), acc[t][i]);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (a.dw) {  // onto the block's weights, which nobody reads any more
                f32x16 o16;
#pragma unroll
                for (int e = 0; e < 16; ++e) o16[e] = 0.f;
#pragma unroll
                for (int t = 0; t < 2 * RT; ++t) {
                    if (t * 16 >= lines) break;
                    const u32x4 xt = few_tr(xs, S, t * 16, f0, lane);
                    o16 = lmfma<DT>(xt, few_row(dzc + l31 * CS + t * 32 + h * 16), o16);
                    if (TWO) o16 = lmfma<DT>(xt, few_row(loc + l31 * CS + t * 32 + h * 16), o16);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<uint2*>(ws + l31 * S + (f0 + 8 * q + 4 * h) * 2) =
                        uint2{lpack2<DT>(o16[4 * q] * os, o16[4 * q + 1] * os), lpack2<DT>(o16[4 * q + 2] * os, o16[4 * q + 3] * os)};
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (a.dw) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < WP; ++i) {
                const int p = lane + 64 * i, v = ch * 32 + p / (FT * 4), at = wave * FT * 4 + p % (FT * 4);
                if (v < a.V && at * 8 < a.d) *reinterpret_cast<u32x4*>(a.dw + v * a.dw_ld + at * 8) = few_row(ws + (p / (FT * 4)) * S + at * 16);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
    if (!a.slab) return;
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < FT; ++i) {
            const int r = t * 32 + l31, f0 = (wave * FT + i) * 32 + 4 * h;
            if (r >= a.N) continue;
            float* dst = a.slab + ((int64_t)blockIdx.x * a.N + r) * a.d;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (f0 + 8 * q < a.d)
                    *reinterpret_cast<f32x4*>(dst + f0 + 8 * q) = f32x4{acc[t][i][4 * q], acc[t][i][4 * q + 1], acc[t][i][4 * q + 2], acc[t][i][4 * q + 3]};
        }
}
// the slices of dx: 32 threads a column of four, every 32nd slice each (with 8 threads the 512 slices of 4 x 21675 x 232 took 7.9 us, so 4.0)
template <int DT>
__global__ __launch_bounds__(256) void class_few_sum_kernel(const float* slab, int slices, int N, int d, uint16_t* out, int64_t ld, const float* outscale) {
    __shared__ f32x4 sm[32][8];
    const int c = (int)threadIdx.x & 7, g = (int)threadIdx.x >> 3, n4 = N * (d / 4), at = (int)blockIdx.x * 8 + c;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (at < n4)
#pragma unroll 8
        for (int s = g; s < slices; s += 32) v += reinterpret_cast<const f32x4*>(slab)[(int64_t)s * n4 + at];
    sm[g][c] = v;
    __syncthreads();
    if (g || at >= n4) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) v += sm[i][c];
    const float os = *outscale;
    const int r = at / (d / 4), f = (at - r * (d / 4)) * 4;
    *reinterpret_cast<uint2*>(out + r * ld + f) = uint2{lpack2<DT>(v[0] * os, v[1] * os), lpack2<DT>(v[2] * os, v[3] * os)};
}

// ---- distillation: the teacher's slots ---------------------------------------------------------------------------------------------------------------
// A workgroup a row, LS lanes a slot (16; 64 for up to 16 slots, whose features would be read one after the other): the student's logits at the teacher's
// classes (dot products in fp32), the teacher's softmax over its filled slots, the loss. Rows of w are fetched from all over the list: 64 (16) of them in
// flight a workgroup, before anything that waits for the row's statistics (1021 x 50 x 512: 13.3 us, behind them 16; 449 x 3 x 920: 7.2, with 16 lanes 9.4).
// saved: [N][1 + 2k] = lse of the row (+inf where the teacher says nothing), logits (log2 units), q -- the first slot that names a class holds the sum over
// all of its slots, the others -1.
__device__ __forceinline__ float row16_sum(float v) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xf, 0xf, true));   // quad_perm [1,0,3,2]
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xf, 0xf, true));   // quad_perm [2,3,0,1]
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xf, 0xf, true));  // row_half_mirror
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xf, 0xf, true));  // row_mirror
}
template <int DT, int LS>
__global__ __launch_bounds__(256) void class_teacher_kernel(const uint16_t* x, int64_t x_ld, const uint16_t* w, int64_t w_ld, const float* off, float c, float coff,
                                                            const int32_t* idx, const void* val, int val_dtype, int k, float itau, float tau2, int N, int V, int d,
                                                            const float* lse, const float* part, int nvb, float* loss, float* saved) {
    __shared__ __attribute__((aligned(16))) int s_idx[512];
    __shared__ __attribute__((aligned(16))) float s_t[512], s_q[512];
    __shared__ float s_z[512], s_sum[4];
    const int t = (int)threadIdx.x, lane = t & 63, wv = t >> 6, r = (int)(blockIdx.y * gridDim.x + blockIdx.x);
    if (r >= N) return;
    const int sub = t / LS, l = t & (LS - 1);
    float* sv = saved + (int64_t)r * (1 + 2 * k);
    const int32_t* ir = idx + (int64_t)r * k;
    // the slots in LDS: class (-1: empty) and the teacher's logit; up to the next four: empty ones
    for (int j = t; j < ((k + 3) & ~3); j += 256) {
        const int v = j < k ? ir[j] : -1;
        s_idx[j] = (unsigned)v < (unsigned)V ? v : -1;
        s_t[j] = j < k ? load_elem(val, (int64_t)r * k + j, val_dtype) * itau : 0.f;
        s_q[j] = 0.f;
    }
    float pm = 0.f, ps = 0.f;
    if (part) {
        if (lane < nvb) {
            pm = part[(int64_t)lane * N + r];
            ps = part[((int64_t)nvb + lane) * N + r];
        }
    } else pm = lse[r];
    __syncthreads();
    constexpr int U = 4;  // slots of LS lanes in flight
    const uint16_t* xr = x + r * x_ld;
    for (int j0 = 0; j0 < k; j0 += 256 / LS * U) {
        float z[U];
        int v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * (256 / LS) + sub;
            v[u] = j < k ? s_idx[j] : -1;
            z[u] = 0.f;
        }
        for (int f = l * 8; f < d; f += LS * 8) {
            const u32x4 xv = *reinterpret_cast<const u32x4*>(xr + f);
            u32x4 wr[U];
#pragma unroll
            for (int u = 0; u < U; ++u) wr[u] = v[u] >= 0 ? *reinterpret_cast<const u32x4*>(w + v[u] * w_ld + f) : u32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    z[u] = fmaf(Elem<DT>::to_f32((uint16_t)(xv[e] & 0xffff)), Elem<DT>::to_f32((uint16_t)(wr[u][e] & 0xffff)), z[u]);
                    z[u] = fmaf(Elem<DT>::to_f32((uint16_t)(xv[e] >> 16)), Elem<DT>::to_f32((uint16_t)(wr[u][e] >> 16)), z[u]);
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * (256 / LS) + sub;
            z[u] = row16_sum(z[u]);
            if (LS == 64) {
                z[u] += __shfl_xor(z[u], 16);
                z[u] += __shfl_xor(z[u], 32);
            }
            if (j < k && l == 0) s_z[j] = z[u];
        }
    }
    float lse_r = pm;
    if (part) {  // few pairs a row: joined here instead of in a launch of their own
        for (int o = 1; o < 64; o *= 2) {
            const float m2 = __shfl_xor(pm, o), s2 = __shfl_xor(ps, o);
            const bool up = lane & o;  // (the same order in every lane: the lower lane's pair first)
            float a0 = up ? m2 : pm, b0 = up ? s2 : ps;
            lse_join(a0, b0, up ? pm : m2, up ? ps : s2);
            pm = a0;
            ps = b0;
        }
        lse_r = ps == 0.f ? -INFINITY : (pm + __builtin_amdgcn_logf(ps)) * kLn2;
    }
    const float l2 = lse_r * kLog2e;
    // the teacher's maximum and sum, by every wave for itself
    float m = -INFINITY, s = 0.f;
    for (int j = lane; j < k; j += 64)
        if (s_idx[j] >= 0) m = m != m || s_t[j] != s_t[j] ? NAN : fmaxf(m, s_t[j]);
    for (int o = 32; o; o >>= 1) {
        const float m2 = __shfl_xor(m, o);
        m = m != m || m2 != m2 ? NAN : fmaxf(m, m2);
    }
    const bool some = m != -INFINITY && l2 != -INFINITY;  // (no filled slot, or nothing but -inf in them, or no class left)
    for (int j = lane; j < k; j += 64)
        if (s_idx[j] >= 0) s += expf(s_t[j] - m);
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    const float ls = logf(s);
    __syncthreads();
    float sum = 0.f;
    for (int j = t; j < k; j += 256) {
        const int v = some ? s_idx[j] : -1;
        float z2 = -INFINITY;
        if (v >= 0) {
            const float ov = off ? class_offset(off[v], coff) : 0.f;
            z2 = ov == -INFINITY ? -INFINITY : fmaf(s_z[j], c, ov);
            const float lq = s_t[j] - m - ls, q = expf(lq);
            if (q != 0.f) sum += q * (lq - (z2 - l2) * kLn2);
            s_q[j] = q;
        }
        sv[1 + j] = z2;
    }
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) s_sum[wv] = sum;
    __syncthreads();
    if (t == 0) {
        loss[r] = some ? (s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3]) * tau2 : 0.f;
        sv[0] = !some ? INFINITY : lse_r == INFINITY ? NAN : lse_r;
    }
    for (int j = t; j < k; j += 256) {
        const int v = s_idx[j];
        float q = s_q[j];
        bool first = some && v >= 0;
        for (int o = 0; o < k; o += 4) {
            const int4 vo = *reinterpret_cast<const int4*>(s_idx + o);
            const f32x4 qo = *reinterpret_cast<const f32x4*>(s_q + o);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool same = (e == 0 ? vo.x : e == 1 ? vo.y : e == 2 ? vo.z : vo.w) == v;
                first = first && !(same && o + e < j);
                q += same && o + e > j ? qo[e] : 0.f;
            }
        }
        sv[1 + k + j] = first ? q : -1.f;
    }
}
// dz at the teacher's classes of a piece (the small tile's launch does it by itself)
template <int DT>
__global__ __launch_bounds__(256) void class_teacher_dz_kernel(const int32_t* idx, const float* saved, const float* lse2, const float* coef, int k, int N, int v_first,
                                                               int Vp, uint16_t* dz, int64_t dz_ld) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)N * k; i += (int64_t)gridDim.x * 256) {
        const int v = idx[i];
        if (v < v_first || v - v_first >= Vp) continue;
        const int r = (int)(i / k), j = (int)(i - (int64_t)r * k);
        TeacherDz t;
        t.load(saved, lse2, coef, k, r, j);
        t.store<DT>(dz + r * dz_ld + (v - v_first));
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------------------
static inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
// 256 x 256 tiles read 131 FLOP per byte staged, 128 x 128 tiles half of that, so the large ones are taken wherever they fill most of the 256 CUs
// (forward with d = 320, large against small: 96 tiles 17.8 us and 13.7, 150 tiles 16.8 and 18.6, 256 tiles 19.1 and 23.0; d = 1024, 130 x 65536 36 and 43) and the
// rows more than half of one (1 x 131072 x 1024: 51 and 44, 128 rows 65 and 61)
static inline bool big_tiles(int64_t rows, int64_t cols) { return rows > 128 && (up(rows, 256) / 256) * (up(cols, 256) / 256) >= 160; }

// The backward's shape: tile, pieces that the class list is cut into, and slices of a piece's classes for dx and of the rows for dw, whose tiles may be few
// (dx: rows x features; dw: classes x features). Times in us, measured: a step of the large tile 0.86, of the small one 0.3 alone on its CU and 0.62 as one of
// two; a tile 6 (8, 5) steps more than its K / 32 (the large one 12 where the two are compared: the estimate is short where
// its tiles are short); a launch is as long as the busiest of an XCD's 32 CUs (64 places), the longer kind of tile first, and 4
// more; slabs of slices move at 4 MB/us.
// dz of a piece stays within 192 MiB, so that it lives in the 256 MiB cache between its three uses -- up to 49152 rows: a piece has at least 2048 classes
// (as far as there are that many), so beyond that dz takes 4 KiB a row and goes through memory, which the estimate does not price.
// 4096 x 65536 x 640: 4 pieces of 4 slices, by equal lengths, took 4 x 219 us for the products, 3 pieces of 5 take 3 x 242. 8400 x 1203 x 1024: dw on 20
// tiles of 8400 rows took 200 us of backward, in 6 slices of the rows 104.
struct GradShape {
    int big, piece, pieces, splits, kper, wsplits, rper, dx_first;
};
static double grad_span(int64_t na, double ta, int64_t nb, double tb, int64_t places) {  // a tiles of ta, then b of tb <= ta
    const int64_t full = na / places, rest = na % places;
    const double t0 = full * ta, t1 = rest ? t0 + ta : t0;  // `rest` places are busy until t1, the others free from t0 on
    if (!nb) return t1;
    const int64_t gap = rest ? (int64_t)(ta / tb) * (places - rest) : 0;
    if (nb > gap) return t1 + (double)((nb - gap + places - 1) / places) * tb;
    return std::max(t1, t0 + (double)((nb + places - rest - 1) / (places - rest)) * tb);
}
static GradShape grad_shape(int64_t N, int64_t V, int64_t d) {
    static const int kCuts[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 14, 16, 20, 24, 32, 48, 64};
    const int64_t rows32 = up(N, 32);
    GradShape best = {}, of_big = {};
    double least = 1e30, least_big = 1e30, more = 0.;  // more: what 6 steps a tile add to of_big
    for (int big = 0; big < 2; ++big) {
        const int64_t bt = big ? 256 : 128;
        const int64_t ntd = up(d, bt) / bt, ntr = up(N, bt) / bt, Vt = up(V, 256) / 256;
        const int64_t most = std::max<int64_t>(8, ((int64_t)96 << 20) / rows32 / 256), n0 = up(Vt, most) / most;  // 256-class tiles of a piece; pieces
        for (int64_t n = n0; n <= 2 * n0 + 2 && n <= Vt; ++n) {
            if (!big && n > 1) break;
            const int64_t pc = up(Vt, n) / n * 256;
            const double logits = n > 1 ? (double)(up(pc / 256 * up(N, 256) / 256, 256) / 256) * (double)(d / 32 + 7) * 0.86 : 0.;
            for (int sw : kCuts) {
                const int64_t rper = up(up(rows32, sw) / sw, 32);
                if (sw > 1 && (rper < 256 || (sw - 1) * rper >= rows32)) break;
                for (int sx : kCuts) {
                    const int64_t kper = up(up(pc, sx) / sx, 32);
                    if (sx > 1 && (kper < 256 || (sx - 1) * kper >= pc)) break;
                    int64_t na = up(pc / bt * ntd * sw, 8) / 8, nb = up(ntr * ntd * sx, 8) / 8;
                    const bool pairs = !big && na + nb > 32;
                    const double step = big ? 0.86 : pairs ? 0.3 + 0.01 * std::min<int64_t>(na + nb - 32, 32) : 0.3, fixed = big ? 6 : pairs ? 5 : 8;
                    const int64_t places = pairs ? 64 : 32;
                    double ta = (rper / 32 + fixed) * step, tb = (kper / 32 + fixed) * step;
                    const bool swap = tb > ta;
                    if (swap) {
                        std::swap(na, nb);
                        std::swap(ta, tb);
                    }
                    const double xslab = n > 1 || sx > 1 ? (double)sx * N * d * 4 / 4e6 : 0., wslab = sw > 1 ? (double)sw * pc * d * 4 / 4e6 : 0.;
                    const double cost = n * (logits + grad_span(na, ta, nb, tb, places) + 4 + xslab * (n > 1 ? 2 : 1) + wslab * 2) + xslab +
                                        (n > 1 ? n * (wslab > 0 ? 4 : 0) + (xslab > 0 ? 4 : 0) : xslab + wslab > 0 ? 4 : 0);
                    if (cost < (big ? least_big : least)) {
                        (big ? least_big : least) = cost;
                        (big ? of_big : best) = GradShape{big, (int)pc, (int)n, sx, (int)kper, sw, (int)rper, swap ? 1 : 0};
                        if (big) more = (double)n * ((na + nb + 31) / 32) * 6 * 0.86;
                    }
                }
            }
        }
    }
    return least_big + more < least ? of_big : best;
}

struct LinPlan {
    bool big_f, direct;  // direct: dx comes out of the one product launch
    int nvb, rows32;
    GradShape g;
    int64_t o_part, o_zlab, o_lse, fwd_bytes;
    int64_t o_lse2, o_coef, o_scale, o_live, o_kept, o_x, o_dz, o_slab, o_wslab, bwd_bytes;
    int few, few_wgs;  // backward of few rows: 0, or row tiles of class_few_kernel; its workgroups (workspace: the scale, 256 bytes, and their slices)
};
// (backward by class_few_kernel and by tiles, V x d = 5000 x 320: 8 rows 11.5 and 23 us, 64 23.3 and 26.1, 96 25.9 and 26.1, 128 28.3 and 26.8; 50000 x 320: 24 and
// 42, 46 and 48, 46.5 and 50.5, 51.3 and 53.3; 365 x 128, 128 rows: 13.4 and 16.4)
static const int kFewRows = 128;
static LinPlan lin_plan(const cdet_linear_loss_desc* q, bool backward) {
    LinPlan p = {};
    const int64_t N = q->N, V = q->V, d = q->d;
    p.big_f = big_tiles(N, V);
    p.nvb = (int)(up(V, p.big_f ? 256 : 128) / (p.big_f ? 128 : 64));
    int64_t o = 0;
    auto take = [&](int64_t bytes) {
        const int64_t at = o;
        o += up(bytes, 256);
        return at;
    };
    p.o_part = take(2 * (int64_t)p.nvb * N * 4);
    p.o_zlab = take(N * 4);
    p.o_lse = take(N * 4);
    p.fwd_bytes = o;
    if (!backward) return p;
    o = 0;
    p.rows32 = (int)up(N, 32);
    // (the last call's shape is kept, by its sizes: the search takes longer than a launch)
    static thread_local int64_t last[3] = {-1, -1, -1};
    static thread_local GradShape shape;
    if (last[0] != N || last[1] != V || last[2] != d) {
        shape = grad_shape(N, V, d);
        last[0] = N;
        last[1] = V;
        last[2] = d;
    }
    p.g = shape;
    p.direct = shape.pieces == 1 && shape.splits == 1;
    p.o_lse2 = take(N * 4);
    p.o_coef = take(N * 4);
    p.o_scale = take(8);
    p.o_live = take(up(N, 256) / 8 + 64);  // (bits; 64 bytes more than they need are read)
    p.o_kept = take(up(V, 256) / 8 + 64);
    p.o_x = p.big_f || shape.big ? take(N * d * 2) : 0;
    p.o_dz = take((int64_t)p.rows32 * shape.piece * 2);
    p.o_slab = p.direct ? 0 : take((int64_t)shape.splits * N * d * 4);
    p.o_wslab = shape.wsplits > 1 ? take((int64_t)shape.wsplits * shape.piece * d * 4) : 0;
    p.bwd_bytes = o;
    if (N <= kFewRows) {
        const int rt = N <= 32 ? 1 : N <= 64 ? 2 : 4, ft = (int)up(up(d, 32) / 32, 8) / 8;
        if (rt * ft <= (rt == 2 ? 6 : rt == 1 ? 4 : 8) && few_lds(rt, (int)N, (int)d) <= 160 * 1024) {
            p.few = rt;
            const double nch = (double)(up(V, 32) / 32);
            const double most = rt * (ft == 3 ? 4 : ft) <= 2 && few_lds(rt, (int)N, (int)d) <= 80 * 1024 ? 512. : 256.;  // two a CU where they fit
            p.few_wgs = (int)std::max(1., std::min(std::min(nch, most), std::sqrt(nch * 1.9e6 / (double)(N * d))));  // (a slice of dx costs what its traffic does)
            p.bwd_bytes = std::max(p.bwd_bytes, 256 + (int64_t)p.few_wgs * N * d * 4);
        }
    }
    return p;
}

static int lin_check(const cdet_linear_loss_desc* q, const char* who) {
    CDET_CHECK_ARG(q, "%s: no descriptor", who);
    CDET_CHECK_ARG(q->dtype == CDET_BF16 || q->dtype == CDET_F16, "%s: x and w must be bf16 or fp16 (dtype %d)", who, q->dtype);
    CDET_CHECK_ARG(q->N >= 0 && q->N <= (1 << 24) && q->V >= 1 && q->V <= (1 << 24), "%s: N %d (0 .. 2^24) or V %d (1 .. 2^24)", who, q->N, q->V);
    CDET_CHECK_ARG(q->d >= 8 && q->d % 8 == 0 && q->d <= 65536, "%s: d = %d must be a multiple of 8 in 8 .. 65536", who, q->d);
    CDET_CHECK_ARG(q->x_ld >= 0 && q->x_ld % 8 == 0 && q->x_ld < (1 << 22) && q->w_ld >= 0 && q->w_ld % 8 == 0 && q->w_ld < (1 << 22),
                   "%s: row pitches %lld, %lld must be multiples of 8 elements below 2^22", who, (long long)q->x_ld, (long long)q->w_ld);
    // (scale / tau and 1 / tau in log2 units, and tau^2, are fp32 numbers)
    CDET_CHECK_ARG(q->tau >= 1e-18f && q->tau <= 1e18f && fabsf(q->scale / q->tau) <= 1e38f, "%s: tau %g (1e-18 .. 1e18) or scale %g (at most 1e38 tau)", who, q->tau, q->scale);
    return 0;
}
static inline bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// a kernel's dynamic LDS above 64 KiB is asked for once per device (`seen`: a bit per device)
template <typename K>
static void allow_lds(std::atomic<uint64_t>& seen, K kernel, size_t bytes) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return;
    const uint64_t bit = 1ull << (dev & 63);
    if (seen.load(std::memory_order_relaxed) & bit) return;
    (void)hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    seen.fetch_or(bit, std::memory_order_relaxed);
}
constexpr size_t LDS_BIG = 4 * 32768, LDS_SMALL = QRING * 16384;

template <bool BWD>
static int launch_logits(LogitArgs a, int dtype, bool big, hipStream_t s) {
    const int bt = big ? 256 : 128;
    a.ntv = div_up(a.V, bt);
    a.ntr = div_up(a.N, bt);
    const int64_t n = (int64_t)a.ntv * a.ntr;
    CDET_CHECK_ARG(n < ((int64_t)1 << 31), "linear loss: too many tiles");
#define CDET_GO(DT_, MT_, NT_, RING_)                                                                      \
    do {                                                                                                   \
        constexpr size_t LDS_ = RING_ + (MT_ == 4 ? 2 * (MT_ * 64 + 4) * 4 : 0);                                                  \
        static std::atomic<uint64_t> seen{0};                                                              \
        allow_lds(seen, class_logits_kernel<DT_, MT_, NT_, BWD>, LDS_);                                    \
        class_logits_kernel<DT_, MT_, NT_, BWD><<<dim3((unsigned)MT_ == 4 ? std::min<int64_t>(n, 256) : n), dim3(kLinThreads<MT_>), LDS_, s>>>(a); \
    } while (0)
    if (dtype == CDET_BF16) {
        if (big) CDET_GO(CDET_BF16, 4, 2, LDS_BIG);
        else CDET_GO(CDET_BF16, 2, 2, LDS_SMALL);
    } else {
        if (big) CDET_GO(CDET_F16, 4, 2, LDS_BIG);
        else CDET_GO(CDET_F16, 2, 2, LDS_SMALL);
    }
#undef CDET_GO
    CDET_LAUNCH_CHECK();
    return 0;
}
static int launch_grads(const GradArgs& a, int dtype, bool big, bool kept, hipStream_t s) {
    const unsigned n = (unsigned)(a.ndw + a.ndx);
#define CDET_GO(DT_, MT_, KEPT_, LDS_)                                                          \
    do {                                                                                        \
        static std::atomic<uint64_t> seen{0};                                                   \
        allow_lds(seen, class_grads_kernel<DT_, MT_, 2, KEPT_>, LDS_);                          \
        class_grads_kernel<DT_, MT_, 2, KEPT_><<<dim3(n), dim3(kLinThreads<MT_>), LDS_, s>>>(a); \
    } while (0)
#define CDET_GRADS(DT_)                                                                         \
    do {                                                                                        \
        if (big && kept) CDET_GO(DT_, 4, true, LDS_BIG);                                        \
        else if (big) CDET_GO(DT_, 4, false, LDS_BIG);                                          \
        else if (kept) CDET_GO(DT_, 2, true, LDS_SMALL);                                        \
        else CDET_GO(DT_, 2, false, LDS_SMALL);                                                 \
    } while (0)
    if (dtype == CDET_BF16) CDET_GRADS(CDET_BF16);
    else CDET_GRADS(CDET_F16);
#undef CDET_GRADS
#undef CDET_GO
    CDET_LAUNCH_CHECK();
    return 0;
}

static int launch_few(const FewArgs& a, int dtype, int rt, int wgs, uint16_t* dx, int64_t dx_ld, hipStream_t s) {
    const size_t lds = (size_t)few_lds(rt, a.N, a.d);
    const int nft = (a.d + 31) / 32;
#define CDET_GO(DT_, RT_, FT_)                                                                        \
    do {                                                                                              \
        static std::atomic<uint64_t> seen{0};                                                         \
        allow_lds(seen, class_few_kernel<DT_, RT_, FT_>, 160 * 1024);                                 \
        class_few_kernel<DT_, RT_, FT_><<<dim3((unsigned)wgs), dim3(512), lds, s>>>(a);               \
    } while (0)
#define CDET_FEW(DT_)                                                                                 \
    do {                                                                                              \
        if (rt == 1) {                                                                                \
            if (nft <= 8) CDET_GO(DT_, 1, 1);                                                         \
            else if (nft <= 16) CDET_GO(DT_, 1, 2);                                                   \
            else CDET_GO(DT_, 1, 4);                                                                  \
        } else if (rt == 2) {                                                                         \
            if (nft <= 8) CDET_GO(DT_, 2, 1);                                                         \
            else CDET_GO(DT_, 2, 3);                                                                  \
        } else {                                                                                      \
            if (nft <= 8) CDET_GO(DT_, 4, 1);                                                         \
            else CDET_GO(DT_, 4, 2);                                                                  \
        }                                                                                             \
    } while (0)
    if (dtype == CDET_BF16) CDET_FEW(CDET_BF16);
    else CDET_FEW(CDET_F16);
#undef CDET_FEW
#undef CDET_GO
    CDET_LAUNCH_CHECK();
    if (!dx) return 0;
    const unsigned nb = (unsigned)div_up((int64_t)a.N * (a.d / 4), 8);
    if (dtype == CDET_BF16) class_few_sum_kernel<CDET_BF16><<<dim3(nb), dim3(256), 0, s>>>(a.slab, wgs, a.N, a.d, dx, dx_ld, a.outscale);
    else class_few_sum_kernel<CDET_F16><<<dim3(nb), dim3(256), 0, s>>>(a.slab, wgs, a.N, a.d, dx, dx_ld, a.outscale);
    CDET_LAUNCH_CHECK();
    return 0;
}

static LogitArgs logit_args(const cdet_linear_loss_desc* q) {
    LogitArgs a = {};
    a.x_ld = q->x_ld;
    a.w_ld = q->w_ld;
    a.c = q->scale / q->tau * kLog2e;
    a.coff = kLog2e / q->tau;
    a.N = q->N;
    a.V = q->V;
    a.d = q->d;
    a.label64 = q->label64;
    return a;
}

// logits' statistics -> lse (and, with labels, the loss); lse null: the statistics only
static int lin_forward(const cdet_linear_loss_desc* q, const LinPlan& p, const void* x, const void* w, const void* label, float* loss, float* lse, char* ws, hipStream_t s) {
    LogitArgs a = logit_args(q);
    a.x = (const uint16_t*)x;
    a.w = (const uint16_t*)w;
    a.off = q->offset;
    a.label = label;
    a.part = (float*)(ws + p.o_part);
    a.zlab = (float*)(ws + p.o_zlab);
    const int rc = launch_logits<false>(a, q->dtype, p.big_f, s);
    if (rc || !lse) return rc;
    int C = 1;  // rows a workgroup: 64 keep the loads wide, fewer fill the chip
    while (C < 64 && (C < 8 ? C < q->N : C * 256 <= q->N)) C *= 2;
    class_lse_kernel<<<dim3(div_up(q->N, C)), dim3(1024), 0, s>>>(a.part, p.nvb, q->N, q->V, C, label, q->label64, a.zlab, loss, lse);
    CDET_LAUNCH_CHECK();
    return 0;
}

static int lin_backward(const cdet_linear_loss_desc* q, const void* x, const void* w, const void* label, const int32_t* idx, const float* saved, int k, const float* lse,
                        int64_t lse_stride, const float* drow, int drow_stride, void* dx, int64_t dx_ld, void* dw, int64_t dw_ld, char* ws, hipStream_t s) {
    const int N = q->N, V = q->V, d = q->d;
    if (!dx && !dw) return 0;
    if (N == 0) {
        if (dw) {
            class_zero_kernel<<<dim3(2048), dim3(256), 0, s>>>((uint16_t*)dw, V, dw_ld, d);
            CDET_LAUNCH_CHECK();
        }
        return 0;
    }
    const LinPlan p = lin_plan(q, true);
    if (p.few && (!idx || N * (int64_t)k <= kFewSlots * 512)) {
        FewArgs a = {};
        a.x = (const uint16_t*)x;
        a.w = (const uint16_t*)w;
        a.x_ld = q->x_ld;
        a.w_ld = q->w_ld;
        a.off = q->offset;
        a.c = q->scale / q->tau * kLog2e;
        a.coff = kLog2e / q->tau;
        a.N = N;
        a.V = V;
        a.d = d;
        a.label = label;
        a.label64 = q->label64;
        a.idx = idx;
        a.saved = saved;
        a.k = k;
        a.lse = lse;
        a.lse_stride = lse_stride;
        a.drow = drow;
        a.drow_stride = drow_stride;
        a.gain = q->scale * (idx ? q->tau : 1.f);
        a.spread = q->dtype == CDET_F16 ? 4096.f : 1.f;
        a.dw = (uint16_t*)dw;
        a.dw_ld = dw_ld;
        a.slab = dx ? (float*)(ws + 256) : nullptr;
        a.outscale = (float*)ws;
        return launch_few(a, q->dtype, p.few, p.few_wgs, (uint16_t*)dx, dx_ld, s);
    }
    float *lse2 = (float*)(ws + p.o_lse2), *coef = (float*)(ws + p.o_coef), *os = (float*)(ws + p.o_scale);
    const float spread = q->dtype == CDET_F16 ? 4096.f : 1.f;
    PrepArgs pa = {};
    pa.drow = drow;
    pa.drow_stride = drow_stride;
    pa.label = label;
    pa.label64 = q->label64;
    pa.lse = lse;
    pa.lse_stride = lse_stride;
    pa.N = N;
    pa.V = V;
    pa.gain = q->scale * (idx ? q->tau : 1.f);
    pa.spread = spread;
    pa.off = q->offset;
    pa.coff = kLog2e / q->tau;
    pa.lse2 = lse2;
    pa.coef = coef;
    pa.outscale = os;
    pa.live = (uint32_t*)(ws + p.o_live);
    pa.kept = (uint32_t*)(ws + p.o_kept);
    pa.x_ld = q->x_ld;
    pa.d8 = d / 8;
    const bool copy_x = p.big_f || p.g.big;
    if (copy_x) {
        pa.x = (const uint16_t*)x;
        pa.xo = (u32x4*)(ws + p.o_x);
    }
    if (N > 32768) {
        class_max_kernel<<<dim3(1), dim3(1024), 0, s>>>(pa, os + 1);
        CDET_LAUNCH_CHECK();
        pa.gmax = os + 1;
    }
    const int64_t most = std::max<int64_t>(std::max(N, V), copy_x ? (int64_t)N * (d / 8) : 0);
    class_prep_kernel<<<dim3((unsigned)std::min<int64_t>(N > 8192 ? 1024 : 256, div_up(most, 1024))), dim3(1024), 0, s>>>(pa);
    CDET_LAUNCH_CHECK();
    const int bt = p.g.big ? 256 : 128;
    SumArgs sum = {};
    sum.d = d;
    sum.outscale = os;
    auto launch_sum = [&](bool sum_dx, bool sum_dw) {
        SumArgs a = sum;
        if (!sum_dx) {  // (the one job comes first)
            a.slab[0] = a.slab[1];
            a.out[0] = a.out[1];
            a.ld[0] = a.ld[1];
            a.rows[0] = a.rows[1];
            a.slices[0] = a.slices[1];
        }
        const int jobs = (sum_dx ? 1 : 0) + (sum_dw ? 1 : 0), rows = jobs == 2 ? std::max(a.rows[0], a.rows[1]) : a.rows[0];
        const dim3 nb((unsigned)std::min<int64_t>(4096, div_up((int64_t)rows * (d / 4), 256)), (unsigned)jobs);
        if (q->dtype == CDET_BF16) class_sum_kernel<CDET_BF16><<<nb, dim3(256), 0, s>>>(a);
        else class_sum_kernel<CDET_F16><<<nb, dim3(256), 0, s>>>(a);
        CDET_LAUNCH_CHECK();
        return 0;
    };
    const bool sum_dx = dx && !p.direct, sum_dw = dw && p.g.wsplits > 1;
    sum.slab[0] = (const float*)(ws + p.o_slab);
    sum.out[0] = (uint16_t*)dx;
    sum.ld[0] = dx_ld;
    sum.rows[0] = N;
    sum.slices[0] = p.g.splits;
    for (int v0 = 0; v0 < V; v0 += p.g.piece) {
        const int Vp = std::min(p.g.piece, V - v0);
        LogitArgs a = logit_args(q);
        a.x = copy_x ? (const uint16_t*)(ws + p.o_x) : (const uint16_t*)x;
        a.x_ld = copy_x ? d : q->x_ld;
        a.w = (const uint16_t*)w + (int64_t)v0 * q->w_ld;
        a.off = q->offset ? q->offset + v0 : nullptr;
        a.live = pa.live;
        a.V = Vp;
        a.label = label;
        a.v_first = v0;
        a.lse2 = lse2;
        a.coef = coef;
        a.dz = (uint16_t*)(ws + p.o_dz);
        a.dz_ld = p.g.piece;
        a.dz_rows = p.rows32;
        // few slots are written by the tile's own workgroup; every tile reads its rows' slots (backward of 997 x 1201 x 320, in the tile and apart: k = 4 26.2 us and
        // 27.8, k = 8 26.7 and 27.6, k = 12 27.6 and 28.0, k = 16 28.7 and 28.3, k = 48 34.0 and 28.7; 200 x 1201 x 64, 1656 x 400 x 160, 500 x 5000 x 256 alike)
        const bool apart = p.big_f || k > 8;
        a.idx = apart ? nullptr : idx;
        a.saved = saved;
        a.k = k;
        int rc = launch_logits<true>(a, q->dtype, p.big_f, s);
        if (rc) return rc;
        if (idx && apart) {
            const unsigned nb = (unsigned)std::min<int64_t>(div_up((int64_t)N * k, 256), 1 << 18);
            if (q->dtype == CDET_BF16) class_teacher_dz_kernel<CDET_BF16><<<dim3(nb), dim3(256), 0, s>>>(idx, saved, lse2, coef, k, N, v0, Vp, a.dz, a.dz_ld);
            else class_teacher_dz_kernel<CDET_F16><<<dim3(nb), dim3(256), 0, s>>>(idx, saved, lse2, coef, k, N, v0, Vp, a.dz, a.dz_ld);
            CDET_LAUNCH_CHECK();
        }
        GradArgs g = {};
        g.x = a.x;
        g.w = a.w;
        g.dz = a.dz;
        g.live = pa.live;
        g.kept = pa.kept + (v0 >> 5);
        g.x_ld = a.x_ld;
        g.w_ld = a.w_ld;
        g.dz_ld = a.dz_ld;
        g.N = N;
        g.rows32 = p.rows32;
        g.d = d;
        g.Vp = Vp;
        g.vk = (int)up(Vp, p.big_f ? 256 : 128);
        g.ntd = div_up(d, bt);
        g.wsplits = p.g.wsplits;
        g.rper = p.g.rper;
        g.wslab = (float*)(ws + p.o_wslab);
        g.ndw = dw ? g.ntd * div_up(Vp, bt) * g.wsplits : 0;
        g.dx_first = p.g.dx_first;
        g.ntr = div_up(N, bt);
        g.kper = p.g.kper;
        g.ndx = dx ? g.ntd * g.ntr * p.g.splits : 0;
        g.dw = dw ? (uint16_t*)dw + (int64_t)v0 * dw_ld : nullptr;
        g.dw_ld = dw_ld;
        g.dx = p.direct ? (uint16_t*)dx : nullptr;
        g.dx_ld = dx_ld;
        g.slab = (float*)(ws + p.o_slab);
        g.add = v0 > 0;
        g.outscale = os;
        rc = launch_grads(g, q->dtype, p.g.big != 0, q->offset != nullptr, s);
        if (rc) return rc;
        const bool ends = v0 + Vp >= V;
        sum.slab[1] = g.wslab;
        sum.out[1] = g.dw;
        sum.ld[1] = dw_ld;
        sum.rows[1] = Vp;
        sum.slices[1] = g.wsplits;
        if (sum_dw || (ends && sum_dx)) rc = launch_sum(ends && sum_dx, sum_dw);
        if (rc) return rc;
    }
    return 0;
}

}  // namespace cdet

using namespace cdet;

extern "C" int64_t cdet_linear_loss_ws_bytes(const cdet_linear_loss_desc* d, int32_t backward) {
    if (!d || d->N <= 0 || d->V <= 0 || d->d <= 0) return 256;
    const LinPlan p = lin_plan(d, backward != 0);
    return backward ? p.bwd_bytes : p.fwd_bytes;
}

#define CDET_LIN_COMMON(who)                                                                                                                          \
    if (int rc__ = lin_check(d, who)) return rc__;                                                                                                    \
    CDET_CHECK_ARG(d->N == 0 || (x && al16(x)), who ": x must be given and 16-byte aligned");                                                           \
    CDET_CHECK_ARG(w && al16(w), who ": w must be given and 16-byte aligned");                                                                          \
    CDET_CHECK_ARG(d->x_ld == 0 || d->x_ld >= d->d, who ": x's row pitch %lld is below d", (long long)d->x_ld);                                         \
    CDET_CHECK_ARG(d->w_ld == 0 || d->w_ld >= d->d, who ": w's row pitch %lld is below d", (long long)d->w_ld);                                         \
    CDET_CHECK_ARG(d->N == 0 || (ws && al16(ws)), who ": the workspace must be given and 16-byte aligned");
#define CDET_LIN_GRADS(who)                                                                                                                            \
    CDET_CHECK_ARG((!dx || (al16(dx) && dx_ld >= d->d && dx_ld % 8 == 0)) && (!dw || (al16(dw) && dw_ld >= d->d && dw_ld % 8 == 0)),                     \
                   who ": dx / dw must be 16-byte aligned with row pitches that are multiples of 8 and at least d");                                   \
    CDET_CHECK_ARG(drow_stride == 0 || drow_stride == 1, who ": drow_stride must be 0 or 1");                                                           \
    CDET_CHECK_ARG((!dx || dx != x) && (!dw || dw != w), who ": dx / dw may not take the place of x / w");

extern "C" int cdet_linear_ce_fwd(const cdet_linear_loss_desc* d, const void* x, const void* w, const void* labels, float* loss, float* lse, void* ws, void* stream) {
    CDET_LIN_COMMON("cdet_linear_ce_fwd")
    CDET_CHECK_ARG(d->tau == 1.f, "cdet_linear_ce_fwd: tau must be 1 (use scale)");
    CDET_CHECK_ARG(d->N == 0 || (labels && loss && lse), "cdet_linear_ce_fwd: labels, loss and lse must be given");
    if (d->N == 0) return 0;
    return lin_forward(d, lin_plan(d, false), x, w, labels, loss, lse, (char*)ws, (hipStream_t)stream);
}

extern "C" int cdet_linear_ce_bwd(const cdet_linear_loss_desc* d, const void* x, const void* w, const void* labels, const float* lse, const float* drow, int32_t drow_stride,
                                  void* dx, int64_t dx_ld, void* dw, int64_t dw_ld, void* ws, void* stream) {
    CDET_LIN_COMMON("cdet_linear_ce_bwd")
    CDET_LIN_GRADS("cdet_linear_ce_bwd")
    CDET_CHECK_ARG(d->tau == 1.f, "cdet_linear_ce_bwd: tau must be 1 (use scale)");
    CDET_CHECK_ARG(d->N == 0 || (labels && lse), "cdet_linear_ce_bwd: labels and lse must be given");
    return lin_backward(d, x, w, labels, nullptr, nullptr, 0, lse, 1, drow, drow_stride, dx, dx_ld, dw, dw_ld, (char*)ws, (hipStream_t)stream);
}

extern "C" int cdet_linear_distill_fwd(const cdet_linear_loss_desc* d, const void* x, const void* w, int32_t k, const int32_t* idx, const void* val, int32_t val_dtype,
                                       float* loss, float* saved, void* ws, void* stream) {
    CDET_LIN_COMMON("cdet_linear_distill_fwd")
    CDET_CHECK_ARG(k >= 1 && k <= 512, "cdet_linear_distill_fwd: k = %d (1 .. 512)", k);
    CDET_CHECK_ARG(val_dtype == CDET_BF16 || val_dtype == CDET_F16 || val_dtype == CDET_F32, "cdet_linear_distill_fwd: val_dtype %d", val_dtype);
    CDET_CHECK_ARG(d->N == 0 || (idx && val && loss && saved), "cdet_linear_distill_fwd: idx, val, loss and saved must be given");
    if (d->N == 0) return 0;
    const LinPlan p = lin_plan(d, false);
    const bool few = p.nvb <= 64;  // (class_teacher_kernel joins them)
    float* lse = few ? nullptr : (float*)((char*)ws + p.o_lse);
    const float* part = few ? (const float*)((char*)ws + p.o_part) : nullptr;
    const int rc = lin_forward(d, p, x, w, nullptr, nullptr, lse, (char*)ws, (hipStream_t)stream);
    if (rc) return rc;
    const dim3 nb((unsigned)std::min(d->N, 1 << 20), (unsigned)div_up(d->N, 1 << 20)), nt(256);  // (a grid's row holds less than 2^32 threads)
    const LogitArgs a = logit_args(d);
#define CDET_GO(DT_, LS_)                                                                                                                                   \
    class_teacher_kernel<DT_, LS_><<<nb, nt, 0, (hipStream_t)stream>>>((const uint16_t*)x, d->x_ld, (const uint16_t*)w, d->w_ld, d->offset, a.c, a.coff, idx, val, val_dtype, \
                                                                 k, 1.f / d->tau, d->tau * d->tau, d->N, d->V, d->d, lse, part, p.nvb, loss, saved)
    // (forward of 6000 x 4000, 64 lanes a slot and 16: d = 320, k = 16 49.1 us and 52.1, k = 24 54.7 and 52.9; d = 192, k = 16 42.5 and 43.1; d = 128, k = 16 39.3 and 37.8)
    const bool wide = k <= 16 && d->d > 128;
    if (d->dtype == CDET_BF16) {
        if (wide) CDET_GO(CDET_BF16, 64);
        else CDET_GO(CDET_BF16, 16);
    } else {
        if (wide) CDET_GO(CDET_F16, 64);
        else CDET_GO(CDET_F16, 16);
    }
#undef CDET_GO
    CDET_LAUNCH_CHECK();
    return 0;
}

extern "C" int cdet_linear_distill_bwd(const cdet_linear_loss_desc* d, const void* x, const void* w, int32_t k, const int32_t* idx, const float* saved, const float* drow,
                                       int32_t drow_stride, void* dx, int64_t dx_ld, void* dw, int64_t dw_ld, void* ws, void* stream) {
    CDET_LIN_COMMON("cdet_linear_distill_bwd")
    CDET_LIN_GRADS("cdet_linear_distill_bwd")
    CDET_CHECK_ARG(k >= 1 && k <= 512, "cdet_linear_distill_bwd: k = %d (1 .. 512)", k);
    CDET_CHECK_ARG(d->N == 0 || (idx && saved), "cdet_linear_distill_bwd: idx and saved must be given");
    return lin_backward(d, x, w, nullptr, idx, saved, k, saved, 1 + 2 * (int64_t)k, drow, drow_stride, dx, dx_ld, dw, dw_ld, (char*)ws, (hipStream_t)stream);
}
