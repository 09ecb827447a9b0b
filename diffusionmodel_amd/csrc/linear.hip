// Linear layer with its epilogue, and its backward pass:
//   z = x W + b + res,  y = act(z);     dz = dy act'(z),  dx = dz W^T,  dW = x^T dz,  db = sum_rows dz
// All three products are C[m, n] = sum_k A(m, k) B(k, n) on one kernel family; an operand is either contiguous along the
// contraction (KC) or along its other index.
#include "blocks.h"
#include "vec.h"
#include <cstdio>
#include <type_traits>

namespace ldm {

namespace {

// The activations, for outputs of type T.  f32 outputs are within 9 half steps of the value (above 2^-119): exponents are
// taken in two parts and reciprocals get a step of Newton's.  For bf16 outputs 2^-11 of the value (GELU: down to -9) is enough,
// and a tile's epilogue has few cycles: the hardware's exp2 and reciprocal as they are, a shorter polynomial.
//
// 1 / d, d >= 1
template <typename T> __device__ __forceinline__ float lin_rcp(float d) {
    const float t = __builtin_amdgcn_rcpf(d);
    return sizeof(T) == 2 ? t : __builtin_fmaf(__builtin_fmaf(-d, t, 1.0f), t, t);
}
// exp(-y), y = hi + lo >= 0 with lo far below hi: exp2 of the rounded product, times 1 + what the rounding left
__device__ __forceinline__ float lin_exp_neg(float hi, float lo) {
    constexpr float c = -1.44269504088896341f, cl = (float)(-1.44269504088896341 - (double)c);
    const float y = hi * c;
    const float r = __builtin_fmaf(hi, cl, __builtin_fmaf(lo, c, __builtin_fmaf(hi, c, -y)));
    const float e = __builtin_amdgcn_exp2f(y);
    return __builtin_fmaf(e * r, 0.69314718055994531f, e);
}
// |z|, at most `most`; NaN stays NaN
__device__ __forceinline__ float lin_abs(float z, float most) {
    const float a = __builtin_fabsf(z);
    return a > most ? most : a;
}
// q = (1 - erf(|z| / sqrt 2)) / 2 and e = exp(-z^2 / 2): q = t poly(t) e with t = 1 / (1 + p |z|), the form of Abramowitz and
// Stegun 7.1.26 with coefficients fitted here (least largest error, by reweighted least squares).  f32: nine terms, off by
// 3.2e-8 of q (4096 x 256 x 1024 with GELU: 27.4 us; five terms off by 1.5e-7 and no corrections: 25.8; without GELU: 24.2).
// bf16: six terms, off by at most 2.5e-8 and, up to |z| = 9, by 2.1e-4 of q, in 12 instructions; the library's erff would cost
// as much as a tile of 256 products.
template <typename T> __device__ __forceinline__ float lin_tail(float z, float& e) {
    if constexpr (sizeof(T) == 2) {
        const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.28f, __builtin_fabsf(z), 1.0f));
        float p = __builtin_fmaf(t, -0.10303881f, 0.37849629f);
        p = __builtin_fmaf(t, p, -0.21841556f);
        p = __builtin_fmaf(t, p, 0.25384381f);
        p = __builtin_fmaf(t, p, 0.07356371f);
        p = __builtin_fmaf(t, p, 0.11555059f);
        const float u = z * 0.84932180028801905f;                                                       // sqrt(log2(e) / 2)
        e = __builtin_amdgcn_exp2f(-u * u);
        return t * p * e;
    } else {
        const float a = lin_abs(z, 64.f), t = lin_rcp<T>(__builtin_fmaf(0.35f, a, 1.0f));
        float p = __builtin_fmaf(t, -0.029108857736f, 0.143787875772f);
        p = __builtin_fmaf(t, p, -0.255326569080f);
        p = __builtin_fmaf(t, p, 0.158721208572f);
        p = __builtin_fmaf(t, p, -0.022790208459f);
        p = __builtin_fmaf(t, p, 0.105368971825f);
        p = __builtin_fmaf(t, p, 0.119869142771f);
        p = __builtin_fmaf(t, p, 0.139856696129f);
        p = __builtin_fmaf(t, p, 0.139621704817f);
        const float h = 0.5f * a, hi = h * a;
        e = lin_exp_neg(hi, __builtin_fmaf(h, a, -hi));
        return t * p * e;
    }
}
// s = 1 / (1 + exp(-z)) and 1 - s
template <typename T> __device__ __forceinline__ float lin_sigmoid(float z, float& rest) {
    if constexpr (sizeof(T) == 2) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504088896341f));
        rest = 1.0f - s;
        return s;
    } else {
        const float e = lin_exp_neg(lin_abs(z, 128.f), 0.f), r = lin_rcp<T>(1.0f + e), er = e * r;
        rest = z < 0.f ? r : er;
        return z < 0.f ? er : r;
    }
}
template <typename T> __device__ __forceinline__ float lin_act(float v, int act) {
    if (act == LIN_SILU) {
        float rest;
        return v * lin_sigmoid<T>(v, rest);
    }
    if (act == LIN_RELU) return v < 0.f ? 0.f : v;
    if (act == LIN_GELU) {
        // v Phi(v) = max(v, 0) - |v| q on either side of zero; q is 0 long before |v| = 64, so infinities give the limits
        float e;
        const float q = lin_tail<T>(v, e);
        return __builtin_fmaf(-__builtin_amdgcn_fmed3f(__builtin_fabsf(v), 0.f, 64.f), q,
                              __builtin_amdgcn_fmed3f(v, 0.f, __builtin_inff()));
    }
    return v;
}
template <typename T> __device__ __forceinline__ float lin_dact(float z, int act) {
    if (act == LIN_SILU) {
        float rest;
        const float s = lin_sigmoid<T>(z, rest);
        return __builtin_fmaf(s * z, rest, s);
    }
    if (act == LIN_RELU) return z > 0.f ? 1.f : 0.f;
    if (act == LIN_GELU) {
        float e;
        const float q = lin_tail<T>(z, e);
        return __builtin_fmaf(z * 0.39894228040143268f, e, z < 0.f ? q : 1.0f - q);
    }
    return 1.f;
}

// ---- the matrix kernel ---------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) computes tiles of TILE x TILE outputs (TILE = 32 F), each wave F x F fragments of
// 16 x 16.  A step of the contraction is 128 bytes of it (64 bf16, 32 f32); NS steps are in LDS, one being read while the
// others arrive.  Both operands keep their memory order in LDS: KC operands as rows of 128 bytes, read by ds_read_b128;
// the others as rows along their contiguous index, read by transposing loads (bf16) or single words (f32).  16-byte
// pieces are XOR-swizzled so that each group of lanes that the LDS serves at once touches every bank once.
//
// The products are taken transposed (first operand = B's columns, second = A's rows), so that a lane's four accumulators
// of a fragment are four consecutive columns of one row.
//
// Per step a wave first multiplies the fragments of the step's first half while it reads those of the second, then waits
// for the next step's data, meets the other waves, and multiplies the second half while it reads the next step's first
// fragments and asks for the step NS later.  One barrier per step; nothing in front of a product is read later than one
// half step before it.
//
// Bound by the matrix cores (256 tile, long contractions: 65536 x 4096 x 1024 bf16 in 443 us = 1.24 PFLOP/s, the rate this
// chip's clock holds under such load; a step alone runs at 1.4), by the epilogue's stores and arithmetic for short ones
// (16384 x 256 x 1024 with GELU and the value before it: 24 us with 128 tiles, 28 with 256, of which the
// products are 7), by LDS reads for the 64 tile.
//
// A wave of the 256 tile has its SIMD for itself and sends an instruction every four cycles or so, 256 in the time of half
// a step's products: what is not a product has to fit between them.  (Walking over several tiles with the requests
// running ahead over a tile's end was measured: its bookkeeping made the step longer than the first loads it hid,
// 497 us against 459 for 65536 x 4096 x 1024.)
// Fragment reads that the compiler does not wait for: GemmFrag::landed() behind an explicit wait makes the values usable.  The
// compiler may not touch such a register in between: tests/test_lds_reads.py looks for that in the built code, and for the
// distances that gemm_mfma_in_place() needs.
template <typename T, bool KC> struct GemmFrag;
template <typename T> struct GemmFrag<T, true> {
    u32x4 v;
    template <int OFF> __device__ __forceinline__ void read(unsigned a) {
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(a), "n"(OFF));
    }
    __device__ __forceinline__ void landed() { asm volatile("" : "+v"(v)); }
    __device__ __forceinline__ u32x4 bits() const { return v; }
    __device__ __forceinline__ float f32(int q) const { return __builtin_bit_cast(f32x4, v)[q]; }
};
template <> struct GemmFrag<__bf16, false> {
    uint2 lo, hi;
    template <int OFF, int NEXT> __device__ __forceinline__ void read(unsigned a) {
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(lo) : "v"(a), "n"(OFF));
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(a), "n"(OFF + NEXT));
    }
    __device__ __forceinline__ void landed() { asm volatile("" : "+v"(lo), "+v"(hi)); }
    __device__ __forceinline__ u32x4 bits() const { return u32x4{lo.x, lo.y, hi.x, hi.y}; }
};
template <> struct GemmFrag<float, false> {
    float q0, q1, q2, q3;
    template <int OFF, int NEXT> __device__ __forceinline__ void read(unsigned a) {
        asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(q0) : "v"(a), "n"(OFF));
        asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(q1) : "v"(a), "n"(OFF + NEXT));
        asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(q2) : "v"(a), "n"(OFF + 2 * NEXT));
        asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(q3) : "v"(a), "n"(OFF + 3 * NEXT));
    }
    __device__ __forceinline__ void landed() { asm volatile("" : "+v"(q0), "+v"(q1), "+v"(q2), "+v"(q3)); }
    __device__ __forceinline__ float f32(int q) const { return q == 0 ? q0 : q == 1 ? q1 : q == 2 ? q2 : q3; }
};

// One operand's tile: where its pieces lie in memory and LDS.
//   KC:   LDS row r (of TILE) holds 128 bytes of the contraction, piece p at slot p ^ ((r >> 1) & 7)
//   else: LDS row k (of BK) holds TILE elements; bf16: 32-byte chunk c at c ^ ((k & 3) + 4 ((k >> 3) & 1)), in rows of only
//         four chunks at c ^ (((k >> 1) & 1) + 2 ((k >> 3) & 1)), of two at c ^ ((k >> 3) & 1); f32: 64-byte chunk c at
//         c ^ ((k >> 2) & 3), in rows of two chunks at c ^ ((k >> 2) & 1)
template <typename T, bool KC, int F> struct GemmOperand {
    static constexpr int ES = sizeof(T), TILE = 32 * F, BK = 128 / ES, BYTES = TILE * 128;
    static constexpr int RB = KC ? 128 : TILE * ES;          // bytes of an LDS row
    static constexpr int NP = BYTES / 4096;                  // pieces per lane and step

    static constexpr int turn(int k) {
        return RB == 64 ? (k >> 3) & 1 : RB == 128 ? ((k >> 1) & 1) | (((k >> 3) & 1) << 1) : (k & 3) | (((k >> 3) & 1) << 2);
    }
    static constexpr int turn32(int k) { return (k >> 2) & (RB == 128 ? 1 : 3); }
    // fragment f (16 rows / columns from w0 + 16 f) of half step s: the address without the parts that are immediate
    static __device__ __forceinline__ unsigned base(int lane, int w0, int s) {
        const int l15 = lane & 15, g = lane >> 4;
        if constexpr (KC) {
            return (w0 + l15) * 128 + (((s * 4 + g) ^ (l15 >> 1)) << 4);
        } else if constexpr (ES == 2) {
            const int row = g * 8 + (l15 >> 2);
            return row * RB + (((w0 >> 4) ^ turn(row)) << 5) + (l15 & 3) * 8;
        } else {
            return (g * 4) * RB + (((w0 >> 4) ^ turn32(g * 4)) << 6) + l15 * 4;
        }
    }
    template <int f, int s> static __device__ __forceinline__ void read(GemmFrag<T, KC>& fr, unsigned b) {
        if constexpr (KC) fr.template read<f * 2048>(b);
        else if constexpr (ES == 2) fr.template read<s * 32 * RB, 4 * RB>(b ^ (f << 5));
        else fr.template read<s * 16 * RB, RB>(b ^ (f << 6));
    }
    // A wave writes 64 consecutive 16-byte slots of the tile at a time.  Lane `lane` of load q of wave w: row
    // first_row(w, lane) + q ROWS, from element(w, q, lane) of that row on.
    static constexpr int ROWS = 1024 / RB;
    static __device__ __forceinline__ int first_row(int w, int lane) { return w * NP * ROWS + lane / (RB / 16); }
    static __device__ __forceinline__ int element(int w, int q, int lane) {
        const int p = lane % (RB / 16), row = w * NP * ROWS + q * ROWS + lane / (RB / 16);
        const int x = KC ? p ^ ((row >> 1) & 7) : ES == 2 ? p ^ (turn(row) << 1) : p ^ (turn32(row) << 2);
        return x * (16 / ES);
    }
};

// v without its first n elements of type T: the rest moved to the front, zeros behind
template <typename T> __device__ __forceinline__ u32x4 gemm_drop(u32x4 v, int n) {
    const int bits = n * (int)sizeof(T) * 8;
    unsigned long long lo = ((unsigned long long)v[1] << 32) | v[0], hi = ((unsigned long long)v[3] << 32) | v[2];
    const unsigned long long l = bits >= 64 ? hi >> (bits & 63) : bits ? (lo >> bits) | (hi << (64 - bits)) : lo;
    const unsigned long long h = bits >= 64 ? 0 : hi >> bits;
    return u32x4{(unsigned)l, (unsigned)(l >> 32), (unsigned)h, (unsigned)(h >> 32)};
}

// the outputs of row m from column n to the last, fewer than eight: residual, the value before the activation, the activation
template <typename T>
__device__ __forceinline__ void gemm_finish(const GemmArgs& a, long m, long n, const float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 7; ++e)
        if (n + e < a.N) {
            float x = v[e];
            if (a.res) x += (float)((const T*)a.res)[m * a.ldr + n + e];
            if (a.pre) ((T*)a.pre)[m * a.ldp + n + e] = (T)x;
            ((T*)a.C)[m * a.ldc + n + e] = (T)lin_act<T>(x, a.act);
        }
}
__device__ __forceinline__ void gemm_bias(const GemmArgs& a, long n, float (&b)[8]) {
    const int left = n >= a.N ? 0 : a.N - n < 8 ? (int)(a.N - n) : 8;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        if (a.bias) row_floats<float>(row_load<float>(a.bias + n + e, left - e), b + e);
        else b[e] = b[e + 1] = b[e + 2] = b[e + 3] = 0.f;
    }
}

// f(0), ..., f(N_ - 1) with the index a constant of the type
template <int I, int N_, typename Fn> __device__ __forceinline__ void gemm_for(Fn&& f) {
    if constexpr (I < N_) {
        f(std::integral_constant<int, I>{});
        gemm_for<I + 1, N_>(f);
    }
}

// 16 bytes per lane from base + lane_off to LDS at dst (of the wave) + 16 lane; offsets from 2^31 on: zeros, no access
__device__ __forceinline__ void gemm_dma(const char* base, char* dst, unsigned lane_off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x80000000, 0x00020000),
                                             (__attribute__((address_space(3))) void*)dst, 16, lane_off, 0, 0, 0);
}
// waits until all but N_ of this wave's memory operations are done (they end in order)
template <int N_> __device__ __forceinline__ void gemm_all_but() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N_ < 63 ? N_ : 63) : "memory");
}
// behind an explicit wait: the compiler takes the value as it stands
template <typename V> __device__ __forceinline__ void gemm_landed(V& v) { asm volatile("" : "+v"(v)); }
// marks v as the one of branch I: branches that pick from a register array by a run-time index stay apart (merged, they
// would make the compiler keep the array in memory)
template <int I, typename V> __device__ __forceinline__ void gemm_pick(V& v) { asm volatile("; %1" : "+v"(v) : "n"(I)); }
// the same for a value in accumulation registers, which LDS takes as they are
template <int I, typename V> __device__ __forceinline__ void gemm_pick_acc(V& v) { asm volatile("; %1" : "+a"(v) : "n"(I)); }
__device__ __forceinline__ void gemm_mfma_in_place(f32x4& c, const u32x4& a, const u32x4& b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// Steps in LDS: the one that is read and those on their way.  A small tile's step is over long before memory answers.
constexpr int gemm_stages(int F, bool dma) { return F == 2 && dma ? 4 : 2; }
constexpr int gemm_lds(int F, bool dma) { return 2 * gemm_stages(F, dma) * F * 4096; }

// DMA: both operands have 16-byte aligned rows whose length along the contiguous index is a multiple of a piece, and come
// by direct loads into LDS.  Otherwise pieces are loaded at element alignment into registers, one (64 tile: two) steps ahead,
// and written to LDS one step before they are read; a piece that would leave its row is taken from the row's end and moved into
// place, so the loads need no branches (which would make the compiler wait for all of them).  That takes rows of at
// least one piece.
template <typename T, bool AKC, bool BKC, int F, bool DMA>
__global__ __launch_bounds__(256, F == 8 ? 1 : 2) void gemm_kernel(GemmArgs a) {
    typedef GemmOperand<T, AKC, F> OA;
    typedef GemmOperand<T, BKC, F> OB;
    constexpr int ES = sizeof(T), V = 16 / ES, TILE = 32 * F, BK = OA::BK, NP = OA::NP, STAGE = OA::BYTES;
    constexpr int NS = gemm_stages(F, DMA);
    typedef typename RowVec<T>::R R;
    constexpr int SETS = !DMA && F == 2 ? 2 : 1;          // register sets in the step loop (two do not fit a tile of 128)
    extern __shared__ __attribute__((aligned(1024))) char smem[];       // [A: NS stages][B: NS stages], then the epilogue's
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

    // the tile: workgroups go round the eight XCDs, and each XCD has a run of neighbouring tiles, in panels of eight columns
    const unsigned per = gridDim.x / 8;
    unsigned lin = blockIdx.x;
    if (lin < per * 8) lin = (lin & 7) * per + (lin >> 3);
    const unsigned ntn = (unsigned)((a.N + TILE - 1) / TILE), ntm = (unsigned)((a.M + TILE - 1) / TILE);
    const unsigned z = lin / (ntn * ntm), id = lin - z * (ntn * ntm);
    const unsigned panel = id / (ntm * 8), in_panel = id - panel * (ntm * 8);
    const unsigned pw = ntn - panel * 8 < 8 ? ntn - panel * 8 : 8;
    const long m0 = (long)(in_panel / pw) * TILE, n0 = (long)(panel * 8 + in_panel % pw) * TILE;
    const long kbeg = (long)z * a.kper * BK;
    const int klen = (int)(a.K - kbeg < (long)a.kper * BK ? a.K - kbeg : (long)a.kper * BK);
    int nt = (klen + BK - 1) / BK;
    if (SETS == 2) nt += nt & 1;          // the register sets take turns: an even number of steps, the last one all zeros
    const int wm = (wave >> 1) * (TILE / 2), wn = (wave & 1) * (TILE / 2);

    // the step that is asked for next, and this lane's pieces of it
    const char* ap = (const char*)a.A + (AKC ? m0 * a.lda + kbeg : kbeg * a.lda + m0) * ES;
    const char* bp = (const char*)a.B + (BKC ? n0 * a.ldb + kbeg : kbeg * a.ldb + n0) * ES;
    const long astep = AKC ? 128 : a.lda * BK * ES, bstep = BKC ? 128 : a.ldb * BK * ES;
    const int arows = (int)(a.M - m0 < (1 << 30) ? a.M - m0 : (1 << 30));      // rows / columns to the end of the matrix
    const int brows = (int)(a.N - n0 < (1 << 30) ? a.N - n0 : (1 << 30));
    int kleft = klen, rstage = 0;
    const int rowa = OA::first_row(wave, lane), rowb = OB::first_row(wave, lane);
    constexpr unsigned NONE = 0x80000000u;
    unsigned va[NP], vb[NP];             // byte offsets from the step's start (through registers: signed)
    // Direct loads: pieces outside the matrix have none.  Through registers: a row no further than the last, a piece no
    // further than the end of its row, which may lie before the step's start (write() moves it into place).  The end of
    // the contraction counts when the last step, or none, is asked for: a branch that two or three steps take, instead of
    // comparisons per piece in all of them.
    auto upto = [](int v, int most) __attribute__((always_inline)) { return v < most ? v : most; };
    auto offsets = [&]() __attribute__((always_inline)) {
        gemm_for<0, NP>([&](auto Q) __attribute__((always_inline)) {
            constexpr int q = Q;
            const int ya = rowa + q * OA::ROWS, xa = OA::element(wave, q, lane);
            const int yb = rowb + q * OB::ROWS, xb = OB::element(wave, q, lane);
            const int enda = AKC ? arows : kleft, enda_x = AKC ? kleft : arows;        // rows, elements of a row
            const int endb = BKC ? brows : kleft, endb_x = BKC ? kleft : brows;
            if constexpr (DMA) {
                va[q] = ya < enda && xa < enda_x ? (unsigned)(ya * (int)a.lda + xa) * ES : NONE;
                vb[q] = yb < endb && xb < endb_x ? (unsigned)(yb * (int)a.ldb + xb) * ES : NONE;
            } else {
                // (nothing left: the first elements of the matrix, which are not used)
                va[q] = kleft > 0 ? (unsigned)((upto(ya, enda - 1) * (int)a.lda + upto(xa, enda_x - V)) * ES) : 0;
                vb[q] = kleft > 0 ? (unsigned)((upto(yb, endb - 1) * (int)a.ldb + upto(xb, endb_x - V)) * ES) : 0;
            }
        });
    };
    auto narrow = [&]() __attribute__((always_inline)) {
        if (kleft < BK) {
            asm volatile("" ::: "memory");
            offsets();
            if (!DMA && kleft <= 0) {
                ap = (const char*)a.A;
                bp = (const char*)a.B;
            }
        }
    };
    u32x4 ra[2][DMA ? 1 : NP], rb[2][DMA ? 1 : NP];
    int rk[2] = {};                       // kleft of the steps in the register sets
    // asks for piece Q of both operands (register set S); behind the last step: zeros, no memory access (DMA), or the
    // first elements of the matrix, which are not used
    auto request = [&](auto Q, auto S) __attribute__((always_inline)) {
        constexpr int q = Q;
        if constexpr (DMA) {
            char* la = smem + rstage * STAGE + (wave * NP + q) * 1024;
            gemm_dma(ap, la, va[q]);
            gemm_dma(bp, la + NS * STAGE, vb[q]);
        } else {
            typedef typename RowVec<T>::V U;
            ra[S][q] = __builtin_bit_cast(u32x4, (R)*(const U*)(ap + (int)va[q]));
            rb[S][q] = __builtin_bit_cast(u32x4, (R)*(const U*)(bp + (int)vb[q]));
        }
    };
    auto requested = [&](auto S) __attribute__((always_inline)) {       // the step is complete: on to the next
        rk[S] = kleft;
        rstage = rstage + 1 == NS ? 0 : rstage + 1;
        kleft -= BK;
        ap += astep;
        bp += bstep;
        narrow();
    };
    // piece Q of register set S is written to stage `st`
    auto put = [&](auto Q, auto S, int st) __attribute__((always_inline)) {
        constexpr int q = Q;
        // taken from the end of its row, or behind the end of k
        if (rk[S] < BK || (!AKC && arows < TILE) || (!BKC && brows < TILE)) {
            const int xa = OA::element(wave, q, lane), xb = OB::element(wave, q, lane);
            const int da = xa - ((AKC ? rk[S] : arows) - V), db = xb - ((BKC ? rk[S] : brows) - V);
            if (da > 0) ra[S][q] = gemm_drop<T>(ra[S][q], da < V ? da : V - 1);
            if (db > 0) rb[S][q] = gemm_drop<T>(rb[S][q], db < V ? db : V - 1);
            if ((AKC ? xa : rowa + q * OA::ROWS) >= rk[S]) ra[S][q] = u32x4{0u, 0u, 0u, 0u};
            if ((BKC ? xb : rowb + q * OB::ROWS) >= rk[S]) rb[S][q] = u32x4{0u, 0u, 0u, 0u};
        }
        char* la = smem + st * STAGE + ((wave * NP + q) * 64 + lane) * 16;
        *(u32x4*)la = ra[S][q];
        *(u32x4*)(la + NS * STAGE) = rb[S][q];
    };

    f32x4 acc[F][F];       // [row fragment][column fragment]
    GemmFrag<T, AKC> fa[2][F];
    GemmFrag<T, BKC> fb[2][F];
    unsigned aa[2], bb[2];      // fragment addresses of the two halves in stage 0, and the stage that is read
    int stage = 0;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        aa[s] = lds0 + OA::base(lane, wm, s);
        bb[s] = lds0 + NS * STAGE + OB::base(lane, wn, s);
    }
    auto landed = [&](auto S) __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
            fa[S][I].landed();
            fb[S][I].landed();
        });
    };
    // products of half H, with the reads of the other half's fragments, and in the second half the requests (register set
    // S), between them
    auto multiply = [&](auto H, auto S) __attribute__((always_inline)) {
        constexpr int h = H, r = 1 - h;
        gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = I;
            if constexpr (h == 1 && i < NP) {
                if constexpr (!DMA) put(I, S, 1 - stage);       // the step after the next, where the last one was
                request(I, S);
            }
            OA::template read<i, r>(fa[r][i], aa[r] + stage * STAGE);
            OB::template read<i, r>(fb[r][i], bb[r] + stage * STAGE);
            gemm_for<0, F>([&](auto J) __attribute__((always_inline)) {
                constexpr int j = J;
                if constexpr (F == 8) {
                    // in place by constraint: with all 256 accumulators live the compiler's own choice moves them about
                    gemm_mfma_in_place(acc[i][j], fb[h][j].bits(), fa[h][i].bits());
                } else if constexpr (ES == 2) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[h][j].bits()),
                                                                        __builtin_bit_cast(bf16x8, fa[h][i].bits()),
                                                                        acc[i][j], 0, 0, 0);
                } else {
                    // lane group g holds k = 4 g .. 4 g + 3; product q takes element q of both operands
                    gemm_for<0, 4>([&](auto Q) __attribute__((always_inline)) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[h][j].f32(Q), fa[h][i].f32(Q), acc[i][j], 0, 0, 0);
                    });
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    // outputs: 32 rows at a time through LDS, so that memory sees whole rows.  One copy of the code for all row fragments
    // (unrolled over them it would not fit the instruction cache), and no load between the stores: loads and stores count
    // together and in order, so a wait for one would be a wait for every store before it (256 x 256 outputs without a
    // residual: 11.7 us with such waits, 6.0 without).
    constexpr int LPR = F * 2, RPP = 64 / LPR, P = 16 / RPP;                       // lanes per row, rows per pass, passes
    constexpr int H = 8 / RowVec<T>::N;                                            // vectors of T in eight columns
    char* tr = smem + wave * 32 * F * 64;
    const int g = lane >> 4, l15 = lane & 15, c = (lane % LPR) * 8, r0 = lane / LPR;
    // slot of 16-byte piece p of row r
    auto slot = [&](int r, int p) __attribute__((always_inline)) { return (r * F * 4 + (p ^ (F == 2 ? r >> 1 : r))) * 16; };
    // G row fragments at a time; RES: with a residual, whose registers leave room for one
    auto finish = [&](auto G_, auto RES) __attribute__((always_inline)) {
        constexpr int G = G_;
        const long n = n0 + wn + c, mw = m0 + wm + r0;
        // the row fragments i .. i + G - 1 (i a multiple of G) go to LDS
        auto spill = [&](int i) __attribute__((always_inline)) {
            gemm_for<0, F / G>([&](auto I) __attribute__((always_inline)) {
                if (i == I * G) gemm_for<0, F * G>([&](auto J) __attribute__((always_inline)) {
                    f32x4 v = acc[I * G + J / F][J % F];
                    if constexpr (F == 8) gemm_pick_acc<I>(v);
                    else gemm_pick<I>(v);
                    *(f32x4*)(tr + J / F * 16 * F * 64 + slot(l15, J % F * 4 + g)) = v;
                });
            });
        };
        // eight columns of pass p (of G P) of them
        auto take = [&](int p, float (&v)[8]) __attribute__((always_inline)) {
            const int r = p % P * RPP + r0;
            const char* t = tr + p / P * 16 * F * 64;
            const f32x4 lo = *(const f32x4*)(t + slot(r, c / 4)), hi = *(const f32x4*)(t + slot(r, c / 4 + 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = lo[e];
                v[4 + e] = hi[e];
            }
        };
        if (!RES && a.part) {
            const long np = (a.N + 7) & ~7L;
            float* part = a.part + (long)z * a.M * np;
#pragma unroll 1
            for (int i = 0; i < F; i += G) {
                spill(i);
                float v[G * P][8];
#pragma unroll
                for (int p = 0; p < G * P; ++p) take(p, v[p]);
#pragma unroll
                for (int p = 0; p < G * P; ++p) {
                    const long m = mw + i * 16 + p * RPP;
                    if (m >= a.M || n >= a.N) continue;
                    *(f32x4*)(part + m * np + n) = f32x4{v[p][0], v[p][1], v[p][2], v[p][3]};
                    *(f32x4*)(part + m * np + n + 4) = f32x4{v[p][4], v[p][5], v[p][6], v[p][7]};
                }
            }
            return;
        }
        const bool full = n + 8 <= a.N;         // else the piece is cut by the last column, or lies behind it
        const int rows = (int)(a.M - m0 < TILE ? a.M - m0 : TILE), rl = wm + r0;
        R res[RES ? F : 1][P * H];
        if constexpr (RES) {
            const char* rp = (const char*)a.res + (m0 * a.ldr + n0) * ES;
            const int ld = (int)a.ldr * ES;
            if (full)
                gemm_for<0, F * P * H>([&](auto I) __attribute__((always_inline)) {
                    constexpr int i = I / (P * H), p = I / H % P, h = I % H;
                    const int r = rl + i * 16 + p * RPP < rows ? rl + i * 16 + p * RPP : rows - 1;
                    res[i][p * H + h] = *(const typename RowVec<T>::V*)(rp + (unsigned)(r * ld + (wn + c) * ES + h * 16));
                });
        }
        if constexpr (RES) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            gemm_for<0, F * P * H>([&](auto I) __attribute__((always_inline)) { gemm_landed(res[I / (P * H)][I % (P * H)]); });
        }
#pragma unroll 1
        for (int i = 0; i < F; i += G) {
            spill(i);
            float v[G * P][8];
#pragma unroll
            for (int p = 0; p < G * P; ++p) take(p, v[p]);
            if constexpr (RES) {
                gemm_for<0, F / G>([&](auto I) __attribute__((always_inline)) {
                    if (i == I * G)
                        gemm_for<0, G * P * H>([&](auto Q) __attribute__((always_inline)) {
                            float r[RowVec<T>::N];
                            R x = res[I * G + Q / (P * H)][Q % (P * H)];
                            gemm_pick<I>(x);
                            row_floats<T>(x, r);
#pragma unroll
                            for (int e = 0; e < RowVec<T>::N; ++e) v[Q / H][(Q % H) * RowVec<T>::N + e] += r[e];
                        });
                });
            }
            auto put = [&](void* out, long ld) __attribute__((always_inline)) {
                char* o = (char*)out + (m0 * ld + n0) * ES;
                const int ldb = (int)ld * ES;
#pragma unroll
                for (int p = 0; p < G * P; ++p)
                    if (full && rl + i * 16 + p * RPP < rows) {
#pragma unroll
                        for (int h = 0; h < H; ++h)
                            row_store<T>((T*)(o + (unsigned)((rl + i * 16 + p * RPP) * ldb + (wn + c) * ES + h * 16)), RowVec<T>::N,
                                         v[p] + h * RowVec<T>::N, ES == 2 && a.through);
                    }
            };
            if (a.pre) put(a.pre, a.ldp);
            auto activate = [&](auto A) __attribute__((always_inline)) {
#pragma unroll
                for (int p = 0; p < G * P; ++p)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[p][e] = lin_act<T>(v[p][e], A);
            };
            if (a.act == LIN_SILU) activate(std::integral_constant<int, LIN_SILU>{});
            else if (a.act == LIN_RELU) activate(std::integral_constant<int, LIN_RELU>{});
            else if (a.act == LIN_GELU) activate(std::integral_constant<int, LIN_GELU>{});
            put(a.C, a.ldc);
            if (n0 + TILE > a.N && (a.N & 7)) {
                // the piece that the last column cuts: element by element
#pragma unroll 1
                for (int p = 0; p < G * P; ++p) {
                    float w[8];
                    take(p, w);
                    const long m = mw + i * 16 + p * RPP;
                    if (m < a.M && n < a.N && !full) gemm_finish<T>(a, m, n, w);
                }
            }
        }
    };

    const std::integral_constant<int, 0> c0;
    const std::integral_constant<int, 1> c1;
    auto ask = [&](auto S) __attribute__((always_inline)) {
        gemm_for<0, NP>([&](auto Q) __attribute__((always_inline)) { request(Q, S); });
        requested(S);
    };
    f32x4 bias[F];
    const int bias_left = a.bias && !a.part ? upto(brows, TILE) : 0;
    gemm_for<0, F>([&](auto J) __attribute__((always_inline)) {
        const int at = wn + J * 16 + (lane >> 4) * 4;
        bias[J] = row_load<float>(a.bias + n0 + at, bias_left - at);
    });
    offsets();
    if constexpr (DMA) {
        for (int t = 0; t < NS; ++t) ask(c0);
        gemm_all_but<(NS - 1) * 2 * NP>();
    } else {
        // the steps 0 and 1 go to LDS; when the loop starts the sets hold the step 2, or 2 and 3
        ask(c0);
        ask(c1);
        gemm_for<0, NP>([&](auto Q) __attribute__((always_inline)) { put(Q, c0, 0); });
        gemm_for<0, NP>([&](auto Q) __attribute__((always_inline)) { put(Q, c1, 1); });
        ask(c0);
        if constexpr (SETS == 2) ask(c1);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // the sums start from the bias (the parts of a split contraction from zero)
    gemm_for<0, F * F>([&](auto I) __attribute__((always_inline)) {
        acc[I / F][I % F] = bias[I % F];
    });
    gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
        OA::template read<I, 0>(fa[0][I], aa[0]);
        OB::template read<I, 0>(fb[0][I], bb[0]);
    });
    landed(c0);
    // a step; S: the register set that holds the one after the next
    auto step = [&](auto S) __attribute__((always_inline)) {
        multiply(c0, S);
        landed(c1);
        const int next = stage + 1 == NS ? 0 : stage + 1;
        // the next step is in LDS: the later ones that were asked for may be on their way (what this wave wrote itself is there
        // since landed())
        if constexpr (DMA) gemm_all_but<(NS - 2) * 2 * NP>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        stage = next;
        multiply(c1, S);
        requested(S);
        landed(c0);
    };
    if constexpr (SETS == 1) {
        for (int t = 0; t < nt; ++t) step(c0);
    } else {
        for (int t = 0; t < nt; t += 2) {
            step(c0);
            step(c1);
        }
    }
    // nothing is on its way into LDS any more, and the last products' results may be read
    gemm_all_but<0>();
    if constexpr (F == 8) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __syncthreads();
    if (a.res && !a.part) finish(std::integral_constant<int, F == 8 || !DMA ? 1 : 2>{}, std::true_type{});
    else finish(std::integral_constant<int, 2>{}, std::false_type{});
}

// Few rows: the weights are read once and that is all there is to do, so the contraction is split over the waves of a
// workgroup and joined in LDS, without a second launch.  A workgroup computes 32 x 32 outputs; its wave w takes the steps
// w, w + 4, ... of the contraction and keeps four of them on the way in LDS of its own, with no barrier before the end.
template <typename T, bool BKC>
__global__ __launch_bounds__(256) void gemm_few_kernel(GemmArgs a) {
    typedef GemmOperand<T, true, 1> OA;
    typedef GemmOperand<T, BKC, 1> OB;
    constexpr int ES = sizeof(T), BK = OA::BK, NS = 4, Q = OA::BYTES / 1024;
    extern __shared__ __attribute__((aligned(1024))) char smem[];       // per wave: [A: NS steps][B: NS steps]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    char* mine = smem + wave * 2 * NS * OA::BYTES;
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)mine;
    const unsigned ntm = (unsigned)((a.M + 31) / 32);
    const long m0 = (long)(blockIdx.x % ntm) * 32, n0 = (long)(blockIdx.x / ntm) * 32;
    const int arows = (int)(a.M - m0 < 32 ? a.M - m0 : 32), brows = (int)(a.N - n0 < 32 ? a.N - n0 : 32);
    const int steps = (int)((a.K + BK - 1) / BK), nt = (steps - wave + 3) / 4;
    const char* ap = (const char*)a.A + m0 * a.lda * ES + wave * 128;
    const char* bp = (const char*)a.B + (BKC ? n0 * a.ldb * ES + wave * 128 : ((long)wave * BK * a.ldb + n0) * ES);
    const long astep = 512, bstep = BKC ? 512 : 4 * a.ldb * BK * ES;
    int kleft = (int)a.K - wave * BK;
    constexpr unsigned NONE = 0x80000000u;
    unsigned va[Q], vb[Q];
    auto offsets = [&]() __attribute__((always_inline)) {
        gemm_for<0, Q>([&](auto I) __attribute__((always_inline)) {
            constexpr int q = I;
            const int ya = OA::first_row(0, lane) + q * OA::ROWS, xa = OA::element(0, q, lane);
            const int yb = OB::first_row(0, lane) + q * OB::ROWS, xb = OB::element(0, q, lane);
            va[q] = ya < arows && xa < kleft ? (unsigned)(ya * (int)a.lda + xa) * ES : NONE;
            vb[q] = yb < (BKC ? brows : kleft) && xb < (BKC ? kleft : brows) ? (unsigned)(yb * (int)a.ldb + xb) * ES : NONE;
        });
    };
    auto request = [&](int t) __attribute__((always_inline)) {
        if (kleft < BK) {
            asm volatile("" ::: "memory");
            offsets();
        }
        char* la = mine + (t & (NS - 1)) * OA::BYTES;
        gemm_for<0, Q>([&](auto I) __attribute__((always_inline)) {
            gemm_dma(ap, la + I * 1024, va[I]);
            gemm_dma(bp, la + NS * OA::BYTES + I * 1024, vb[I]);
        });
        kleft -= 4 * BK;
        ap += astep;
        bp += bstep;
    };
    f32x4 acc[2][2] = {};                 // [row fragment][column fragment]
    GemmFrag<T, true> fa[2][2];
    GemmFrag<T, BKC> fb[2][2];
    const unsigned aa[2] = {lds0 + OA::base(lane, 0, 0), lds0 + OA::base(lane, 0, 1)};
    const unsigned bb[2] = {lds0 + NS * OA::BYTES + OB::base(lane, 0, 0), lds0 + NS * OA::BYTES + OB::base(lane, 0, 1)};
    offsets();
    for (int t = 0; t < NS; ++t) request(t);
    for (int t = 0; t < nt; ++t) {
        gemm_all_but<(NS - 1) * 2 * Q>();
        const unsigned st = (t & (NS - 1)) * OA::BYTES;
        gemm_for<0, 2>([&](auto S) __attribute__((always_inline)) {
            gemm_for<0, 2>([&](auto I) __attribute__((always_inline)) {
                OA::template read<I, S>(fa[S][I], aa[S] + st);
                OB::template read<I, S>(fb[S][I], bb[S] + st);
            });
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        gemm_for<0, 2>([&](auto S) __attribute__((always_inline)) {
            gemm_for<0, 2>([&](auto I) __attribute__((always_inline)) {
                fa[S][I].landed();
                fb[S][I].landed();
            });
        });
        request(t + NS);
        gemm_for<0, 8>([&](auto I) __attribute__((always_inline)) {
            constexpr int h = I / 4, i = I / 2 % 2, j = I % 2;
            if constexpr (ES == 2) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[h][j].bits()),
                                                                    __builtin_bit_cast(bf16x8, fa[h][i].bits()), acc[i][j], 0, 0, 0);
            } else {
                gemm_for<0, 4>([&](auto E) __attribute__((always_inline)) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[h][j].f32(E), fa[h][i].f32(E), acc[i][j], 0, 0, 0);
                });
            }
        });
    }
    gemm_all_but<0>();                    // nothing is on its way into LDS any more
    __syncthreads();
    // the waves' sums, 32 x 32 each (rows of 36 floats), then four columns per thread
    float* join = (float*)smem;
    constexpr int ROW = 36;
    const int g = lane >> 4, l15 = lane & 15;
    gemm_for<0, 4>([&](auto I) __attribute__((always_inline)) {
        constexpr int i = I / 2, j = I % 2;
        *(f32x4*)(join + (wave * 32 + i * 16 + l15) * ROW + j * 16 + g * 4) = acc[i][j];
    });
    __syncthreads();
    const int r = tid / 8, c = (tid % 8) * 4, left = brows - c;
    if (r >= arows || left <= 0) return;
    const long m = m0 + r, n = n0 + c;
    float v[4];
    row_floats<float>(row_load<float>(a.bias + n, a.bias ? left : 0), v);
    for (int w = 0; w < 4; ++w) {
        const f32x4 p = *(const f32x4*)(join + (w * 32 + r) * ROW + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) {
            if (a.res) v[e] += (float)((const T*)a.res)[m * a.ldr + n + e];
            if (a.pre) ((T*)a.pre)[m * a.ldp + n + e] = (T)v[e];
            ((T*)a.C)[m * a.ldc + n + e] = (T)lin_act<T>(v[e], a.act);
        }
}

// Any sizes, strides and alignment, element by element: 64 x 64 outputs per workgroup, 64 bytes of the contraction per step.
// Serves the products with an operand whose rows are shorter than one 16-byte piece.
constexpr int GT = 64, GROW = 64 + 16;      // bytes of an LDS row: 64 of data, padded against bank conflicts
template <typename T, bool AKC, bool BKC>
__global__ __launch_bounds__(256) void gemm_any_kernel(GemmArgs a) {
    constexpr int ES = sizeof(T), KB = 64 / ES;
    __shared__ __attribute__((aligned(16))) char As[GT * GROW];
    __shared__ __attribute__((aligned(16))) char Bs[GT * GROW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = lane >> 4, l15 = lane & 15;
    const unsigned ntn = (unsigned)((a.N + GT - 1) / GT), ntm = (unsigned)((a.M + GT - 1) / GT);
    const unsigned z = blockIdx.x / (ntn * ntm), id = blockIdx.x - z * (ntn * ntm);
    const long m0 = (long)(id / ntn) * GT, n0 = (long)(id % ntn) * GT;
    const long kbeg = (long)z * a.kper * 2 * KB, kmost = kbeg + (long)a.kper * 2 * KB, kend = a.K < kmost ? a.K : kmost;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    f32x4 acc[2][2] = {};      // [n][m]
    for (long k0 = kbeg; k0 < kend; k0 += KB) {
        __syncthreads();
        for (int i = tid; i < GT * KB; i += 256) {
            const int r = AKC ? i / KB : i % GT, k = AKC ? i % KB : i / GT;
            T v = (T)0.f;
            if (m0 + r < a.M && k0 + k < kend) v = ((const T*)a.A)[AKC ? (m0 + r) * a.lda + k0 + k : (k0 + k) * a.lda + m0 + r];
            *(T*)(As + r * GROW + k * ES) = v;
        }
        for (int i = tid; i < GT * KB; i += 256) {
            const int r = BKC ? i / KB : i % GT, k = BKC ? i % KB : i / GT;
            T v = (T)0.f;
            if (n0 + r < a.N && k0 + k < kend) v = ((const T*)a.B)[BKC ? (n0 + r) * a.ldb + k0 + k : (k0 + k) * a.ldb + n0 + r];
            *(T*)(Bs + r * GROW + k * ES) = v;
        }
        __syncthreads();
        u32x4 fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = *(const u32x4*)(As + (wm + i * 16 + l15) * GROW + g * 16);
            fb[i] = *(const u32x4*)(Bs + (wn + i * 16 + l15) * GROW + g * 16);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (ES == 2) {
                    acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[j]),
                                                                        __builtin_bit_cast(bf16x8, fa[i]), acc[j][i], 0, 0, 0);
                } else {
                    const f32x4 va = __builtin_bit_cast(f32x4, fa[i]), vb = __builtin_bit_cast(f32x4, fb[j]);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vb[q], va[q], acc[j][i], 0, 0, 0);
                }
            }
    }
    const long np = (a.N + 7) & ~7L;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long m = m0 + wm + i * 16 + l15;
        if (m >= a.M) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const long n = n0 + wn + j * 16 + g * 4 + r;
                if (n >= a.N) continue;
                float v = acc[j][i][r];
                if (a.part) {
                    a.part[((long)z * a.M + m) * np + n] = v;
                    continue;
                }
                if (a.bias) v += a.bias[n];
                if (a.res) v += (float)((const T*)a.res)[m * a.ldr + n];
                if (a.pre) ((T*)a.pre)[m * a.ldp + n] = (T)v;
                ((T*)a.C)[m * a.ldc + n] = (T)lin_act<T>(v, a.act);
            }
    }
}

// joins the parts of a split contraction, in order, and finishes: outputs 8 i .. 8 i + 7
template <typename T>
__device__ __forceinline__ void gemm_join(const GemmArgs& a, int parts, long i) {
    constexpr int V = RowVec<T>::N;
    const long np = (a.N + 7) & ~7L, pieces = np / 8;
    if (i >= a.M * pieces) return;
    const long m = i / pieces, n = (i - m * pieces) * 8;
    const int left = a.N - n < 8 ? (int)(a.N - n) : 8;
    float v[8];
    gemm_bias(a, n, v);
    const float* p = a.part + m * np + n;
    float s[8] = {};
    for (int z = 0; z < parts; ++z, p += a.M * np) {
        const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            s[e] += lo[e];
            s[4 + e] += hi[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += s[e];
#pragma unroll
    for (int h = 0; h < 8; h += V) {
        if (a.res) {
            float r[V];
            row_floats<T>(row_load<T>((const T*)a.res + m * a.ldr + n + h, left - h), r);
#pragma unroll
            for (int e = 0; e < V; ++e) v[h + e] += r[e];
        }
        if (a.pre) row_store<T>((T*)a.pre + m * a.ldp + n + h, left - h, v + h);
#pragma unroll
        for (int e = 0; e < V; ++e) v[h + e] = lin_act<T>(v[h + e], a.act);
        row_store<T>((T*)a.C + m * a.ldc + n + h, left - h, v + h);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a, int parts) {
    gemm_join<T>(a, parts, (long)blockIdx.x * 256 + threadIdx.x);
}

// What the backward pass leaves for its end, in one launch (each costs some 4 us): the joins of dx and dw, and the bias
// gradient's sums over the dz kernel's workgroups, 16 threads per column, in a fixed order.
// 1001 x 321 -> 643 f32: 47.1 us with three launches, 39.8 with one; 16384 x 1024 -> 4096 bf16: the same within 1 %
template <typename T>
__global__ __launch_bounds__(256) void linear_finish_kernel(GemmArgs x, int xparts, unsigned xblocks, GemmArgs w, int wparts,
                                                            unsigned sblocks, const float* part, int G, long N, float* db) {
    if (blockIdx.x >= sblocks) {
        const unsigned b = blockIdx.x - sblocks;
        if (b < xblocks) gemm_join<T>(x, xparts, (long)b * 256 + threadIdx.x);
        else gemm_join<T>(w, wparts, (long)(b - xblocks) * 256 + threadIdx.x);
        return;
    }
    __shared__ float sm[16][17];
    const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4;
    const long c = (long)blockIdx.x * 16 + cl;
    float s = 0.f;
    if (c < N) {
#pragma unroll 8
        for (int g = sl; g < G; g += 16) s += part[g * N + c];
    }
    sm[sl][cl] = s;
    __syncthreads();
    if (sl == 0 && c < N) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += sm[i][cl];
        db[c] = t;
    }
}

// dz = dy act'(pre), and the column sums of dz over this workgroup's rows (part [gridDim.x][N]).  dz is rounded to the element
// type: bf16 is what the matrix cores multiply, and dz is the caller's gradient of `res`.  The products of a bf16 call are then
// off by 0.0023 in norm, where the rounding of their own outputs alone gives 0.0017; two bf16 parts of dz would double both
// products' time.  The column sums take it unrounded.
// One pass over dy and pre and one write, bound by HBM: a thread keeps eight (f32: four) columns, `ct` threads cover a row's
// part, 256 / ct rows go at once, and each thread asks for four rows before it uses the first.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T* dy, long lddy, const T* pre, long ldp, T* dz, long lddz,
                                                        float* part, long M, long N, int act, int ct) {
    constexpr int V = RowVec<T>::N, U = 4;
    __shared__ float join[256 * V];
    const int c = threadIdx.x % ct, rg = threadIdx.x / ct, rgs = 256 / ct;
    const long n = ((long)blockIdx.y * ct + c) * V;
    const int left = n >= N ? 0 : N - n < V ? (int)(N - n) : V;
    const long step = (long)gridDim.x * rgs;
    float s[V] = {};
    for (long m = (long)blockIdx.x * rgs + rg; m < M; m += U * step) {
        typename RowVec<T>::R vd[U], vp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = m + u * step;
            vd[u] = row_load<T>(dy + r * lddy + n, r < M ? left : 0);
            if (act != LIN_NONE) vp[u] = row_load<T>(pre + r * ldp + n, r < M ? left : 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long r = m + u * step;
            float v[V];
            row_floats<T>(vd[u], v);
            if (act != LIN_NONE) {
                float p[V];
                row_floats<T>(vp[u], p);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] *= lin_dact<T>(p[e], act);
                row_store<T>(dz + r * lddz + n, r < M ? left : 0, v);
            }
            if (r < M) {
#pragma unroll
                for (int e = 0; e < V; ++e) s[e] += v[e];
            }
        }
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < V; ++e) join[threadIdx.x * V + e] = s[e];
    __syncthreads();
    for (int i = threadIdx.x; i < ct * V; i += 256) {
        float t = 0.f;
        for (int j = 0; j < rgs; ++j) t += join[j * ct * V + i];
        const long col = (long)blockIdx.y * ct * V + i;
        if (col < N) part[blockIdx.x * N + col] = t;
    }
}

// Tile and split of one product: the pair with the least estimated time.  The estimate is what the kernels measured (us):
// a workgroup costs `fixed` (first loads, epilogue) and per step of the contraction `busy` where several share a CU and hide
// each other's waits, `lone` where one has a CU for itself; a split adds a launch and the traffic of its f32 parts.
//   bf16, 16384 x 1024 outputs of K = 1024:  tiles of 256: 36.2 us, 128: 38.7, 64: 69.7      (K = 256: 17.3, 17.8, 35.0)
//   bf16,  1024 x 1024 outputs of K = 2048:  128: 25.7 us, in two parts 19.8; 64: 11.3, in two parts 18.2
//   bf16,   256 x 1024 outputs of K = 16384: 128: 142.5 us whole, 25.7 in sixteen parts; 64: 55.6 whole, 22.0 in four
// f32 steps are bound by their matrix instructions, a sixteenth of bf16's rate; operands staged through registers cost
// about twice the direct loads' step.
struct GemmPlan { int F, parts, kper; };
struct GemmCost { int F; double fixed, busy, lone; };
constexpr GemmCost kBf16Direct[3] = {{8, 11.0, 1.5, 1.5}, {4, 2.5, 0.45, 0.60}, {2, 1.7, 0.17, 0.25}};
constexpr GemmCost kBf16Staged[2] = {{4, 3.4, 0.80, 1.20}, {2, 1.7, 0.34, 0.50}};
constexpr GemmCost kF32[2] = {{4, 4.0, 1.90, 2.0}, {2, 1.8, 0.50, 0.55}};
// `extra`: what a tile's epilogue adds
double gemm_us(const GemmCost& c, long M, long N, long parts, long kper, double extra) {
    const long t = 32 * c.F, per_cu = (((M + t - 1) / t) * ((N + t - 1) / t) * parts + 255) / 256;
    return per_cu <= 1 ? c.fixed + kper * c.lone + extra : per_cu * (c.fixed + kper * c.busy + extra);
}
GemmPlan gemm_plan(int es, long M, long N, long K, bool dma) {
    const GemmCost* costs = es == 4 ? kF32 : dma ? kBf16Direct : kBf16Staged;
    const int n = es == 2 && dma ? 3 : 2;
    const long bk = 128 / es, steps = K > 0 ? (K + bk - 1) / bk : 1;
    GemmPlan best = {2, 1, (int)steps};
    double least = 1e30;
    for (int i = 0; i < n; ++i) {
        const long t = 32 * costs[i].F, tiles = ((M + t - 1) / t) * ((N + t - 1) / t);
        for (long want = 1; want <= 64 && want <= steps; ++want) {
            const long kper = (steps + want - 1) / want, parts = (steps + kper - 1) / kper;
            double us = gemm_us(costs[i], M, N, parts, kper, 0.0);
            if (parts > 1) us += 4.0 + (double)M * N * (8.0 * parts + es) / 7e6;
            if (us < least) {
                least = us;
                best = {costs[i].F, (int)parts, (int)kper};
            }
            if (tiles * parts >= 1024) break;       // more parts only add traffic
        }
    }
    return best;
}
// The tile of a whole bf16 product with an epilogue: a workgroup of the 256 tile has its CU for itself and nothing to
// multiply meanwhile; two of the 128 tile hide one's epilogue behind the other's products, as long as what they write stays
// in the caches.  us per tile of (256, 128, 64), outputs written through / larger ones:
//   GELU 8.0, 1.1, 0.15   SiLU 3.0, 0.45, 0.05   residual 7.0, 1.2, 0.3 / 10, 2.2, 0.5   z kept 2.5, 0.3, 0.05 / 5.2, 2.3, 0.5
//   16384 x 256 x 1024: GELU and z kept 27.7 us with the 256 tile, 23.6 with 128; 65536 x 256 x 1024: 109.6, 118.3, GELU
//   alone 92.9, 78.0; residual 105.1, 100.1
int gemm_tile_with_epilogue(const GemmArgs& a, int steps) {
    static constexpr double gelu[3] = {8.0, 1.1, 0.15}, silu[3] = {3.0, 0.45, 0.05};
    static constexpr double res[2][3] = {{7.0, 1.2, 0.3}, {10.0, 2.2, 0.5}}, pre[2][3] = {{2.5, 0.3, 0.05}, {5.2, 2.3, 0.5}};
    const int large = !a.through;
    int F = 8;
    double least = 1e30;
    for (int i = 0; i < 3; ++i) {
        const double extra = (a.act == LIN_GELU ? gelu[i] : a.act == LIN_SILU ? silu[i] : 0.0) + (a.res ? res[large][i] : 0.0) +
                             (a.pre ? pre[large][i] : 0.0);
        const double us = gemm_us(kBf16Direct[i], a.M, a.N, 1, steps, extra);
        if (us < least) {
            least = us;
            F = kBf16Direct[i].F;
        }
    }
    return F;
}
long gemm_part_floats(const GemmPlan& p, long M, long N) { return p.parts > 1 ? p.parts * M * ((N + 7) & ~7L) : 0; }

// what ldm_last_kernel() says of a product
#define GEMM_BOOL(b) ((b) ? "true" : "false")
#define GEMM_TYPE(T) (sizeof(T) == 2 ? "bf16" : "f32")
template <typename T, bool AKC, bool BKC, int F, bool DMA>
const char* gemm_name() {
    static char name[64];
    static const int n = snprintf(name, sizeof name, "gemm_kernel<%s, %s, %s, %d, %s>", GEMM_TYPE(T), GEMM_BOOL(AKC), GEMM_BOOL(BKC), F,
                                  GEMM_BOOL(DMA));
    (void)n;
    return name;
}
template <typename T, bool BKC>
const char* gemm_few_name() {
    static char name[64];
    static const int n = snprintf(name, sizeof name, "gemm_few_kernel<%s, %s>", GEMM_TYPE(T), GEMM_BOOL(BKC));
    (void)n;
    return name;
}
template <typename T, bool AKC, bool BKC>
const char* gemm_any_name() {
    static char name[64];
    static const int n = snprintf(name, sizeof name, "gemm_any_kernel<%s, %s, %s>", GEMM_TYPE(T), GEMM_BOOL(AKC), GEMM_BOOL(BKC));
    (void)n;
    return name;
}

template <typename T, bool AKC, bool BKC, int F, bool DMA>
int gemm_launch(const GemmArgs& a, unsigned grid, hipStream_t s) {
    static bool done[kMaxDevices] = {};
    LDM_TRY(allow_dynamic_lds((const void*)&gemm_kernel<T, AKC, BKC, F, DMA>, gemm_lds(F, DMA), done));
    set_last_kernel(gemm_name<T, AKC, BKC, F, DMA>());
    gemm_kernel<T, AKC, BKC, F, DMA><<<grid, 256, gemm_lds(F, DMA), s>>>(a);
    LDM_HIP(hipGetLastError());
    return LDM_OK;
}

// products for gemm_few_kernel: up to 64 rows, and in bf16 at most 16 MB of weights, whose rows it reads in pieces of 64
// bytes (us, against the 64 tile; [K, N] weights): 4 rows bf16 2048 x 256: 5.6 / 12.9, 1024 x 1024: 6.0 / 6.7, 4096 x 4096:
// 20.0 / 12.0; f32 2048 x 256: 13.0 / 21.5, 4096 x 4096: 23.2 / 27.4.  The rule does not look at the length of the contraction,
// which only its four waves share: 32 x 262144 x 32 takes 284 us.
bool gemm_is_few(int es, long M, long N, long K) { return M <= 64 && (es == 4 || K * N <= (1L << 23)); }

constexpr long kMostTiles = 1L << 24;      // a launch holds less than 2^32 threads

template <typename T, bool AKC, bool BKC>
int gemm(GemmArgs a, float* ws, GemmJoin* later, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return LDM_OK;
    // the stride of a single row is never used, whatever it is
    if (a.M == 1) a.ldc = a.ldr = a.ldp = 0;
    if ((AKC ? a.M : a.K) == 1) a.lda = 0;
    if ((BKC ? a.N : a.K) == 1) a.ldb = 0;
    constexpr long V = 16 / sizeof(T);
    const long alen = AKC ? a.K : a.M, blen = BKC ? a.K : a.N;          // elements of an operand's row
    auto aligned = [&](const void* p, long ld, long len) { return (size_t)p % 16 == 0 && ld % V == 0 && len % V == 0; };
    const bool dma = aligned(a.A, a.lda, alen) && aligned(a.B, a.ldb, blen);
    // the kernel's offsets within a tile are 32 bits
    constexpr long most = 1L << 21;
    LDM_REQUIRE(a.lda <= most && a.ldb <= most && a.ldc <= most && (!a.res || a.ldr <= most) && (!a.pre || a.ldp <= most),
                "rows of a matrix are more than 2^21 elements apart");
    if constexpr (AKC)
        if (dma && gemm_is_few(sizeof(T), a.M, a.N, a.K)) {
            static bool done[kMaxDevices] = {};
            constexpr int lds = 4 * 2 * 4 * 4096;
            LDM_TRY(allow_dynamic_lds((const void*)&gemm_few_kernel<T, BKC>, lds, done));
            const long grid = (a.M + 31) / 32 * ((a.N + 31) / 32);
            LDM_REQUIRE(grid < kMostTiles, "more output tiles than one launch holds");
            set_last_kernel(gemm_few_name<T, BKC>());
            gemm_few_kernel<T, BKC><<<(unsigned)grid, 256, lds, s>>>(a);
            LDM_HIP(hipGetLastError());
            return LDM_OK;
        }
    // bf16: a lane's eight columns are one access, and a row's lanes cover whole lines
    a.through = sizeof(T) == 2 && a.M * a.N * (a.pre ? 4 : 2) <= kThroughBytes && a.N % 64 == 0 && a.ldc % 64 == 0 &&
                (size_t)a.C % 128 == 0 && (!a.pre || (a.ldp % 64 == 0 && (size_t)a.pre % 128 == 0));
    GemmPlan p = gemm_plan(sizeof(T), a.M, a.N, a.K, dma);
    if (sizeof(T) == 2 && dma && p.parts == 1 && (a.act != LIN_NONE || a.res || a.pre)) p.F = gemm_tile_with_epilogue(a, p.kper);
    LDM_REQUIRE(p.parts == 1 || ws, "this product needs a workspace");
    // rows too short for a piece, or an empty contraction, which has no row at all to read
    const bool any = a.K == 0 || alen < V || blen < V;
    const long t = any ? GT : 32 * p.F, tiles = ((a.M + t - 1) / t) * ((a.N + t - 1) / t) * p.parts;
    LDM_REQUIRE(tiles < kMostTiles, "more output tiles than one launch holds");
    LDM_REQUIRE(a.K / p.parts < (1L << 30), "a contraction longer than 2^30");
    a.kper = p.kper;
    a.part = p.parts > 1 ? ws : nullptr;
    if (any) {
        set_last_kernel(gemm_any_name<T, AKC, BKC>());
        gemm_any_kernel<T, AKC, BKC><<<(unsigned)tiles, 256, 0, s>>>(a);
        LDM_HIP(hipGetLastError());
    } else if (!dma && p.F == 2) LDM_TRY((gemm_launch<T, AKC, BKC, 2, false>(a, (unsigned)tiles, s)));
    else if (!dma) LDM_TRY((gemm_launch<T, AKC, BKC, 4, false>(a, (unsigned)tiles, s)));
    else if (p.F == 2) LDM_TRY((gemm_launch<T, AKC, BKC, 2, true>(a, (unsigned)tiles, s)));
    else if (p.F == 4) LDM_TRY((gemm_launch<T, AKC, BKC, 4, true>(a, (unsigned)tiles, s)));
    else if constexpr (sizeof(T) == 2) LDM_TRY((gemm_launch<T, AKC, BKC, 8, true>(a, (unsigned)tiles, s)));
    if (p.parts > 1) {
        const long n = a.M * ((a.N + 7) / 8);
        const unsigned blocks = (unsigned)((n + 255) / 256);
        if (later) {
            *later = {a, p.parts, blocks};
            return LDM_OK;
        }
        gemm_join_kernel<T><<<blocks, 256, 0, s>>>(a, p.parts);
        LDM_HIP(hipGetLastError());
    }
    return LDM_OK;
}
template <typename T>
int gemm_by_order(const GemmArgs& a, bool akc, bool bkc, float* ws, GemmJoin* later, hipStream_t s) {
    return akc ? (bkc ? gemm<T, true, true>(a, ws, later, s) : gemm<T, true, false>(a, ws, later, s))
               : gemm<T, false, false>(a, ws, later, s);
}

// threads per row of the dz kernel, workgroups along the rows (at least four rows a thread where there are that many; one,
// whose sums need no second launch, up to sixteen) and along the columns
struct DzShape { int ct; long groups, blocks; };
DzShape dz_shape(int es, long M, long N) {
    const long nvec = (N * es + 15) / 16;
    DzShape d;
    d.ct = 1;
    while (d.ct < 256 && d.ct < nvec) d.ct *= 2;
    d.blocks = (nvec + d.ct - 1) / d.ct;
    if (M == 0) return {d.ct, 0, d.blocks};
    const long rows = (M + 256 / d.ct - 1) / (256 / d.ct);
    d.groups = rows <= 16 ? 1 : (rows + 3) / 4;
    const long most = d.blocks < 1024 ? 1024 / d.blocks : 1;
    if (d.groups > most) d.groups = most;
    return d;
}

}  // namespace

int launch_gemm(int dtype, const GemmArgs& a, bool akc, bool bkc, float* ws, GemmJoin* later, hipStream_t s) {
    return dtype == LDM_BF16 ? gemm_by_order<__bf16>(a, akc, bkc, ws, later, s)
                             : gemm_by_order<float>(a, akc, bkc, ws, later, s);
}

long gemm_ws_floats(int dtype, long M, long N, long K) {
    // which tile it will be depends on the alignment as well
    long n = 0;
    for (int dma = 0; dma < 2; ++dma) {
        const long f = gemm_part_floats(gemm_plan(dtype == LDM_BF16 ? 2 : 4, M, N, K, dma), M, N);
        n = f > n ? f : n;
    }
    return n;
}

long linear_dz_ws_floats(int dtype, long M, long N) { return dz_shape(dtype == LDM_BF16 ? 2 : 4, M, N).groups * N; }

template <typename T>
static int dz_launch(const void* dy, long lddy, const void* pre, long ldp, void* dz, long lddz, float* db, float* ws, long M,
                     long N, int act, int* groups, hipStream_t s) {
    const DzShape d = dz_shape(sizeof(T), M, N);
    LDM_REQUIRE(d.blocks <= 65535, "too many columns for one launch");
    const bool direct = d.groups == 1;          // the one partial row is the result
    *groups = !db || direct ? -1 : (int)d.groups;
    if (M > 0 && (act != LIN_NONE || db)) {
        linear_dz_kernel<T><<<dim3((unsigned)d.groups, (unsigned)d.blocks), 256, 0, s>>>(
            (const T*)dy, lddy, (const T*)pre, ldp, (T*)dz, lddz, direct ? db : db ? ws : nullptr, M, N, act, d.ct);
        LDM_HIP(hipGetLastError());
    }
    return LDM_OK;
}
int launch_linear_dz(int dtype, const void* dy, long lddy, const void* pre, long ldp, void* dz, long lddz, float* db, float* ws,
                     long M, long N, int act, int* groups, hipStream_t s) {
    return dtype == LDM_BF16 ? dz_launch<__bf16>(dy, lddy, pre, ldp, dz, lddz, db, ws, M, N, act, groups, s)
                             : dz_launch<float>(dy, lddy, pre, ldp, dz, lddz, db, ws, M, N, act, groups, s);
}
int launch_linear_finish(int dtype, const GemmJoin& x, const GemmJoin& w, const float* part, int groups, long N, float* db,
                         hipStream_t s) {
    const unsigned sblocks = groups >= 0 ? (unsigned)((N + 15) / 16) : 0, grid = sblocks + x.blocks + w.blocks;
    if (grid == 0) return LDM_OK;
    if (dtype == LDM_BF16)
        linear_finish_kernel<__bf16><<<grid, 256, 0, s>>>(x.a, x.parts, x.blocks, w.a, w.parts, sblocks, part, groups, N, db);
    else linear_finish_kernel<float><<<grid, 256, 0, s>>>(x.a, x.parts, x.blocks, w.a, w.parts, sblocks, part, groups, N, db);
    LDM_HIP(hipGetLastError());
    return LDM_OK;
}

}  // namespace ldm
