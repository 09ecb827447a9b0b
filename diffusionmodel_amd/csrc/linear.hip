// Linear layer with its epilogue, and its backward pass:
//   z = x W + b + res,  y = act(z);     dz = dy act'(z),  dx = dz W^T,  dW = x^T dz,  db = sum_rows dz
// All three products are C[m, n] = sum_k A(m, k) B(k, n) on one kernel family; an operand is either contiguous along the
// contraction (KC) or along its other index.
#include "blocks.h"
#include "vec.h"
#include <type_traits>

namespace ldm {

namespace {

// exp and the reciprocal by the hardware's instructions (one step of f32 each)
__device__ __forceinline__ float lin_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and e = exp(-z^2 / 2): Abramowitz and Stegun 7.1.26, erfc(x) = poly(t) exp(-x^2) with
// t = 1 / (1 + 0.3275911 x), off by at most 1.5e-7; the negative side takes erfc itself, without 1 - ...  A tile's epilogue
// has few cycles for this: 12 instructions, where the library's erff would cost as much as a tile of 256 products.
__device__ __forceinline__ float lin_phi(float z, float& e) {
    const float x = __builtin_fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.0f));
    float p = __builtin_fmaf(t, 1.061405429f, -1.453152027f);
    p = __builtin_fmaf(t, p, 1.421413741f);
    p = __builtin_fmaf(t, p, -0.284496736f);
    p = __builtin_fmaf(t, p, 0.254829592f);
    e = lin_exp(-x * x);
    const float tail = 0.5f * t * p * e;
    return z >= 0.f ? 1.0f - tail : tail;
}
__device__ __forceinline__ float lin_act(float v, int act) {
    if (act == LIN_SILU) return v * __builtin_amdgcn_rcpf(1.0f + lin_exp(-v));
    if (act == LIN_RELU) return v < 0.f ? 0.f : v;
    if (act == LIN_GELU) {
        float e;
        return v * lin_phi(v, e);
    }
    return v;
}
__device__ __forceinline__ float lin_dact(float z, int act) {
    if (act == LIN_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + lin_exp(-z));
        return s * (1.0f + z * (1.0f - s));
    }
    if (act == LIN_RELU) return z > 0.f ? 1.f : 0.f;
    if (act == LIN_GELU) {
        float e;
        const float phi = lin_phi(z, e);
        return __builtin_fmaf(z * 0.39894228040143268f, e, phi);
    }
    return 1.f;
}

// ---- the matrix kernel ---------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) computes a tile of TILE x TILE outputs (TILE = 32 F), each wave F x F fragments of
// 16 x 16.  A step of the contraction is 128 bytes of it (64 bf16, 32 f32); two steps are staged in LDS, one being read
// while the other arrives.  Both operands keep their memory order in LDS: KC operands as rows of 128 bytes, read by
// ds_read_b128; the others as rows along their contiguous index, read by transposing loads (bf16) or single words (f32).
// 16-byte pieces are XOR-swizzled so that each group of lanes that the LDS serves at once touches every bank once.
//
// The products are taken transposed (first operand = B's columns, second = A's rows), so that a lane's four accumulators
// of a fragment are four consecutive columns of one row.
//
// Per step a wave first multiplies the fragments of the step's first half while it reads those of the second, then waits
// for the next step's data, meets the other waves, and multiplies the second half while it reads the next step's first
// fragments and asks for the step after it.  One barrier per step; nothing in front of a product is read later than one
// half step before it.
// Fragment reads that the compiler does not wait for: GemmFrag::landed() behind an explicit wait makes the values usable.
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
//         four chunks at c ^ (((k >> 1) & 1) + 2 ((k >> 3) & 1)); f32: 64-byte chunk c at c ^ ((k >> 2) & 3)
template <typename T, bool KC, int F> struct GemmOperand {
    static constexpr int ES = sizeof(T), TILE = 32 * F, BK = 128 / ES, BYTES = TILE * 128;
    static constexpr int RB = KC ? 128 : TILE * ES;          // bytes of an LDS row
    static constexpr int NP = BYTES / 4096;                  // pieces per lane and step

    static constexpr int turn(int k) {
        return RB == 128 ? ((k >> 1) & 1) | (((k >> 3) & 1) << 1) : (k & 3) | (((k >> 3) & 1) << 2);
    }
    // fragment f (16 rows / columns from w0 + 16 f) of half step s: the address without the parts that are immediate
    static __device__ __forceinline__ unsigned base(int lane, int w0, int s) {
        const int l15 = lane & 15, g = lane >> 4;
        if constexpr (KC) {
            return (w0 + l15) * 128 + (((s * 4 + g) ^ (l15 >> 1)) << 4);
        } else if constexpr (ES == 2) {
            const int row = g * 8 + (l15 >> 2);
            return row * RB + (((w0 >> 4) ^ turn(row)) << 5) + (l15 & 3) * 8;
        } else {
            return (g * 4) * RB + (((w0 >> 4) ^ g) << 6) + l15 * 4;
        }
    }
    template <int f, int s> static __device__ __forceinline__ void read(GemmFrag<T, KC>& fr, unsigned b) {
        if constexpr (KC) fr.template read<f * 2048>(b);
        else if constexpr (ES == 2) fr.template read<s * 32 * RB, 4 * RB>(b ^ (f << 5));
        else fr.template read<s * 16 * RB, RB>(b ^ (f << 6));
    }
    // the piece of memory that goes to 16-byte slot `slot` of the tile: row of the tile and element within the row
    static __device__ __forceinline__ void piece(int slot, int& row, int& el) {
        row = slot / (RB / 16);
        const int p = slot % (RB / 16);
        int q;
        if constexpr (KC) q = p ^ ((row >> 1) & 7);
        else if constexpr (ES == 2) q = p ^ (turn(row) << 1);
        else q = p ^ (((row >> 2) & 3) << 2);
        el = q * (16 / ES);
    }
};

// the first n of 16 / sizeof(T) elements at p (element aligned), zeros for the rest; n may be zero or less, or more than all
typedef u32x4 gemm_u16_a2 __attribute__((aligned(2)));
typedef u32x4 gemm_u16_a4 __attribute__((aligned(4)));
template <typename T> __device__ __forceinline__ u32x4 gemm_guarded(const T* p, int n) {
    constexpr int N = 16 / sizeof(T);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (n >= N) {
        if constexpr (sizeof(T) == 2) v = *(const gemm_u16_a2*)p;
        else v = *(const gemm_u16_a4*)p;
    } else if (n > 0) {
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
            if (e < n) {
                if constexpr (sizeof(T) == 2) v[e >> 1] |= (unsigned)((const unsigned short*)p)[e] << ((e & 1) * 16);
                else v[e] = ((const unsigned*)p)[e];
            }
    }
    return v;
}

// 8 outputs of row m from column n on: bias, residual, the value before the activation, the activation
template <typename T>
__device__ __forceinline__ void gemm_finish(const GemmArgs& a, long m, long n, float (&v)[8], const float (&bias)[8]) {
    typedef T VT __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    typedef float VF __attribute__((ext_vector_type(8)));
    const bool full = n + 8 <= a.N;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias[e];
    if (a.res) {
        const T* r = (const T*)a.res + m * a.ldr + n;
        if (full) {
            const VF f = __builtin_convertvector(*(const VT*)r, VF);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += f[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < a.N) v[e] += (float)r[e];
        }
    }
    VF o;
    if (a.pre) {
        T* p = (T*)a.pre + m * a.ldp + n;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[e];
        if (full) {
            *(VT*)p = __builtin_convertvector(o, VT);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (n + e < a.N) p[e] = (T)v[e];
        }
    }
    T* c = (T*)a.C + m * a.ldc + n;
    if (a.act == LIN_SILU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lin_act(v[e], LIN_SILU);
    } else if (a.act == LIN_RELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lin_act(v[e], LIN_RELU);
    } else if (a.act == LIN_GELU) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = lin_act(v[e], LIN_GELU);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = v[e];
    if (full) {
        *(VT*)c = __builtin_convertvector(o, VT);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (n + e < a.N) c[e] = (T)v[e];
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

// behind an explicit wait: the compiler takes the value as it stands
template <typename V> __device__ __forceinline__ void gemm_landed(V& v) { asm volatile("" : "+v"(v)); }
// marks v as the one of branch I: branches that pick from a register array by a run-time index stay apart (merged, they
// would make the compiler keep the array in memory)
template <int I, typename V> __device__ __forceinline__ void gemm_pick(V& v) { asm volatile("; %1" : "+v"(v) : "n"(I)); }
__device__ __forceinline__ void gemm_mfma_in_place(f32x4& c, const u32x4& a, const u32x4& b) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}

// Steps in LDS: the one that is read and those on their way.  A small tile's step is over long before memory answers.
constexpr int gemm_stages(int F, bool dma) { return F == 2 && dma ? 4 : 2; }

// DMA: both operands have 16-byte aligned rows whose length along the contiguous index is a multiple of a piece, and come
// by direct loads into LDS; otherwise they are staged through registers, with every access guarded.
template <typename T, bool AKC, bool BKC, int F, bool DMA>
__global__ __launch_bounds__(256, F == 8 ? 1 : 2) void gemm_kernel(GemmArgs a) {
    typedef GemmOperand<T, AKC, F> OA;
    typedef GemmOperand<T, BKC, F> OB;
    constexpr int ES = sizeof(T), TILE = 32 * F, BK = OA::BK, NP = OA::NP, STAGE = OA::BYTES, NS = gemm_stages(F, DMA);
    extern __shared__ __attribute__((aligned(1024))) char smem[];       // [A: NS stages][B: NS stages]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;

    // the tile: neighbouring tiles on one XCD (workgroups go round the eight XCDs), panels of eight tile columns
    const unsigned total = gridDim.x, per = total / 8;
    unsigned lin = blockIdx.x;
    if (lin < per * 8) lin = (lin & 7) * per + (lin >> 3);
    const unsigned ntn = (unsigned)((a.N + TILE - 1) / TILE), ntm = (unsigned)((a.M + TILE - 1) / TILE);
    const unsigned z = lin / (ntn * ntm), id = lin - z * (ntn * ntm);
    const unsigned panel = id / (ntm * 8), in_panel = id - panel * (ntm * 8);
    const unsigned pw = ntn - panel * 8 < 8 ? ntn - panel * 8 : 8;
    const long m0 = (long)(in_panel / pw) * TILE, n0 = (long)(panel * 8 + in_panel % pw) * TILE;
    const long kbeg = (long)z * a.kper * BK, kend = a.K < kbeg + (long)a.kper * BK ? a.K : kbeg + (long)a.kper * BK;
    const int nt = (int)((kend - kbeg + BK - 1) / BK);

    const int wm = (wave >> 1) * (TILE / 2), wn = (wave & 1) * (TILE / 2);
    const char* ap = (const char*)a.A + (AKC ? m0 * a.lda + kbeg : kbeg * a.lda + m0) * ES;
    const char* bp = (const char*)a.B + (BKC ? n0 * a.ldb + kbeg : kbeg * a.ldb + n0) * ES;
    const long astep = AKC ? 128 : a.lda * BK * ES, bstep = BKC ? 128 : a.ldb * BK * ES;
    const int arows = (int)(a.M - m0 < TILE ? a.M - m0 : TILE), brows = (int)(a.N - n0 < TILE ? a.N - n0 : TILE);
    const int klen = (int)(kend - kbeg < (1L << 30) ? kend - kbeg : (1L << 30));

    // this lane's pieces: offset from the step's start (out of range where the tile ends), and index along k
    constexpr unsigned NONE = 0x80000000u;
    unsigned va[NP], vb[NP];
    int ka[NP], kb[NP], ea[NP], eb[NP];
#pragma unroll
    for (int q = 0; q < NP; ++q) {
        int row, el;
        OA::piece((wave * NP + q) * 64 + lane, row, el);
        const int ma = AKC ? row : el;
        ka[q] = AKC ? el : row;
        ea[q] = el;
        va[q] = ma < arows ? (unsigned)((long)row * a.lda * ES + el * ES) : NONE;
        OB::piece((wave * NP + q) * 64 + lane, row, el);
        const int mb = BKC ? row : el;
        kb[q] = BKC ? el : row;
        eb[q] = el;
        vb[q] = mb < brows ? (unsigned)((long)row * a.ldb * ES + el * ES) : NONE;
    }
    u32x4 ra[DMA ? 1 : NP], rb[DMA ? 1 : NP];
    // asks for piece q of both operands of step t (steps behind the last one: zeros, without a memory access)
    auto request = [&](int t, int q) __attribute__((always_inline)) {
        const int kleft = klen - t * BK;
        if constexpr (DMA) {
            const auto sa = __builtin_amdgcn_make_buffer_rsrc((void*)(ap + t * astep), 0, 0x80000000, 0x00020000);
            const auto sb = __builtin_amdgcn_make_buffer_rsrc((void*)(bp + t * bstep), 0, 0x80000000, 0x00020000);
            char* la = smem + (t % NS) * STAGE + (wave * NP + q) * 1024;
            const unsigned oa = kleft < BK && ka[q] >= kleft ? NONE : va[q], ob = kleft < BK && kb[q] >= kleft ? NONE : vb[q];
            __builtin_amdgcn_raw_ptr_buffer_load_lds(sa, (__attribute__((address_space(3))) void*)la, 16, oa, 0, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(sb, (__attribute__((address_space(3))) void*)(la + NS * STAGE), 16, ob, 0, 0, 0);
        } else {
            ra[q] = gemm_guarded<T>((const T*)(ap + t * astep + va[q]),
                                    va[q] == NONE || ka[q] >= kleft ? 0 : AKC ? kleft - ka[q] : arows - ea[q]);
            rb[q] = gemm_guarded<T>((const T*)(bp + t * bstep + vb[q]),
                                    vb[q] == NONE || kb[q] >= kleft ? 0 : BKC ? kleft - kb[q] : brows - eb[q]);
        }
    };
    // step t's pieces of this wave are in LDS (requests of later steps may still be on their way: they count in order)
    auto land = [&](int t) __attribute__((always_inline)) {
        if constexpr (DMA) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * 2 * NP) : "memory");
        } else {
            char* la = smem + (t % NS) * STAGE + (wave * NP * 64 + lane) * 16;
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                *(u32x4*)(la + q * 1024) = ra[q];
                *(u32x4*)(la + NS * STAGE + q * 1024) = rb[q];
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    };

    f32x4 acc[F][F];       // [row fragment][column fragment]
    gemm_for<0, F * F>([&](auto I) __attribute__((always_inline)) { acc[I / F][I % F] = f32x4{0.f, 0.f, 0.f, 0.f}; });
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
    // products of half S, with the reads of the other half's fragments (and a step's requests) between them
    auto multiply = [&](auto S, auto REQ, int t) __attribute__((always_inline)) {
        constexpr int s = S, r = 1 - S;
        gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = I;
            if constexpr (REQ) {
                if constexpr (i < NP) request(t + NS, i);
            }
            OA::template read<i, r>(fa[r][i], aa[r] + stage * STAGE);
            OB::template read<i, r>(fb[r][i], bb[r] + stage * STAGE);
            gemm_for<0, F>([&](auto J) __attribute__((always_inline)) {
                constexpr int j = J;
                if constexpr (F == 8) {
                    // in place by constraint: with all 256 accumulators live the compiler's own choice moves them about
                    gemm_mfma_in_place(acc[i][j], fb[s][j].bits(), fa[s][i].bits());
                } else if constexpr (ES == 2) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[s][j].bits()),
                                                                        __builtin_bit_cast(bf16x8, fa[s][i].bits()),
                                                                        acc[i][j], 0, 0, 0);
                } else {
                    gemm_for<0, 4>([&](auto Q) __attribute__((always_inline)) {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[s][j].f32(Q), fa[s][i].f32(Q), acc[i][j], 0, 0, 0);
                    });
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto step = [&](int t) __attribute__((always_inline)) {
        multiply(std::integral_constant<int, 0>{}, std::false_type{}, t);
        landed(std::integral_constant<int, 1>{});
        land(t + 1);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        stage = stage + 1 == NS ? 0 : stage + 1;
        multiply(std::integral_constant<int, 1>{}, std::true_type{}, t);
        landed(std::integral_constant<int, 0>{});
    };

    if (nt > 0) {
        if constexpr (DMA) {
#pragma unroll
            for (int t = 0; t < NS; ++t)
#pragma unroll
                for (int q = 0; q < NP; ++q) request(t, q);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * 2 * NP) : "memory");
        } else {
#pragma unroll
            for (int q = 0; q < NP; ++q) request(0, q);
            land(0);
#pragma unroll
            for (int q = 0; q < NP; ++q) request(1, q);
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
            OA::template read<I, 0>(fa[0][I], aa[0]);
            OB::template read<I, 0>(fb[0][I], bb[0]);
        });
        landed(std::integral_constant<int, 0>{});
        for (int t = 0; t < nt; ++t) step(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");            // nothing is on its way into LDS any more
    }
    // the last products' results may be read
    if constexpr (F == 8) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __syncthreads();

    // epilogue: 16 rows at a time through LDS, so that memory sees whole rows.  One copy of the code for all row fragments
    // (unrolled over them it would not fit the instruction cache), and no load between the stores: loads and stores count
    // together and in order, so a wait for one would be a wait for every store before it (256 x 256 outputs without a
    // residual: 11.7 us with such waits, _EPI_ without).
    constexpr int ROW = F * 64 + 16, LPR = F * 2, RPP = 64 / LPR, P = 16 / RPP;     // bytes of a row, lanes per row, rows
    typedef typename RowVec<T>::R R;                                               // per pass, passes
    constexpr int H = 16 / RowVec<T>::N / 2;                                       // vectors of T in eight columns
    char* tr = smem + wave * 16 * ROW;
    const int g = lane >> 4, l15 = lane & 15, c = (lane % LPR) * 8, r0 = lane / LPR;
    const long n = n0 + wn + c, mw = m0 + wm + r0;
    auto spill = [&](int i) __attribute__((always_inline)) {
        gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
            if (i == I) gemm_for<0, F>([&](auto J) __attribute__((always_inline)) {
                f32x4 v = acc[I][J];
                gemm_pick<I>(v);
                *(f32x4*)(tr + l15 * ROW + J * 64 + g * 16) = v;
            });
        });
    };
    auto take = [&](int p, float (&v)[8]) {
        const f32x4 lo = *(const f32x4*)(tr + (p * RPP + r0) * ROW + c * 4), hi = *(const f32x4*)(tr + (p * RPP + r0) * ROW + c * 4 + 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = lo[e];
            v[4 + e] = hi[e];
        }
    };
    if (a.part) {
        const long np = (a.N + 7) & ~7L;
        float* part = a.part + (long)z * a.M * np;
#pragma unroll 1
        for (int i = 0; i < F; ++i) {
            spill(i);
            float v[P][8];
#pragma unroll
            for (int p = 0; p < P; ++p) take(p, v[p]);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const long m = mw + i * 16 + p * RPP;
                if (m >= a.M || n >= a.N) continue;
                *(f32x4*)(part + m * np + n) = f32x4{v[p][0], v[p][1], v[p][2], v[p][3]};
                *(f32x4*)(part + m * np + n + 4) = f32x4{v[p][4], v[p][5], v[p][6], v[p][7]};
            }
        }
        return;
    }
    float bias[8];
    gemm_bias(a, n, bias);
    if (n0 + TILE > a.N) {
        // the last tile column, where a piece of eight may be cut: guarded, piece by piece
#pragma unroll 1
        for (int i = 0; i < F; ++i) {
            spill(i);
#pragma unroll 1
            for (int p = 0; p < P; ++p) {
                float v[8];
                take(p, v);
                const long m = mw + i * 16 + p * RPP;
                if (m < a.M && n < a.N) gemm_finish<T>(a, m, n, v, bias);
            }
        }
        return;
    }
    R res[F][P * H];
    if (a.res) {
        gemm_for<0, F * P * H>([&](auto I) __attribute__((always_inline)) {
            constexpr int i = I / (P * H), p = I / H % P, h = I % H;
            const long m = mw + i * 16 + p * RPP < a.M ? mw + i * 16 + p * RPP : a.M - 1;
            res[i][p * H + h] = *(const typename RowVec<T>::V*)((const T*)a.res + m * a.ldr + n + h * RowVec<T>::N);
        });
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    gemm_for<0, 8>([&](auto E) __attribute__((always_inline)) { gemm_landed(bias[E]); });
    if (a.res) gemm_for<0, F * P * H>([&](auto I) __attribute__((always_inline)) { gemm_landed(res[I / (P * H)][I % (P * H)]); });
#pragma unroll 1
    for (int i = 0; i < F; ++i) {
        spill(i);
        float v[P][8];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            take(p, v[p]);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[p][e] += bias[e];
        }
        if (a.res) {
            gemm_for<0, F>([&](auto I) __attribute__((always_inline)) {
                if (i == I)
                    gemm_for<0, P * H>([&](auto Q) __attribute__((always_inline)) {
                        float r[RowVec<T>::N];
                        R x = res[I][Q];
                        gemm_pick<I>(x);
                        row_floats<T>(x, r);
#pragma unroll
                        for (int e = 0; e < RowVec<T>::N; ++e) v[Q / H][(Q % H) * RowVec<T>::N + e] += r[e];
                    });
            });
        }
        const long m = mw + i * 16;
        auto put = [&](T* out, long ld) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < P; ++p)
                if (m + p * RPP < a.M) {
#pragma unroll
                    for (int h = 0; h < H; ++h)
                        row_store<T>(out + (m + p * RPP) * ld + n + h * RowVec<T>::N, RowVec<T>::N, v[p] + h * RowVec<T>::N);
                }
        };
        if (a.pre) put((T*)a.pre, a.ldp);
        auto activate = [&](auto A) __attribute__((always_inline)) {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[p][e] = lin_act(v[p][e], A);
        };
        if (a.act == LIN_SILU) activate(std::integral_constant<int, LIN_SILU>{});
        else if (a.act == LIN_RELU) activate(std::integral_constant<int, LIN_RELU>{});
        else if (a.act == LIN_GELU) activate(std::integral_constant<int, LIN_GELU>{});
        put((T*)a.C, a.ldc);
    }
}

// joins the parts of a split contraction, in order, and finishes
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(GemmArgs a, int parts) {
    const long np = (a.N + 7) & ~7L, pieces = np / 8;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.M * pieces) return;
    const long m = i / pieces, n = (i - m * pieces) * 8;
    float bias[8], v[8] = {};
    gemm_bias(a, n, bias);
    const float* p = a.part + m * np + n;
    for (int z = 0; z < parts; ++z, p += a.M * np) {
        const f32x4 lo = *(const f32x4*)p, hi = *(const f32x4*)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] += lo[e];
            v[4 + e] += hi[e];
        }
    }
    gemm_finish<T>(a, m, n, v, bias);
}

// dz = dy act'(pre), and the column sums of dz over this workgroup's rows (part [gridDim.x][N]).  One pass over dy and pre
// and one write, bound by HBM: a thread keeps eight (f32: four) columns, `ct` threads cover a row's part, 256 / ct rows go
// at once, and each thread asks for four rows before it uses the first.
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
                for (int e = 0; e < V; ++e) v[e] *= lin_dact(p[e], act);
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
//   bf16, 16384 x 1024 outputs of K = 1024:  tiles of 256: 38.3 us, 128: 40.5, 64: 69.0      (K = 256: 21.2, 21.2, 38.0)
//   bf16,  1024 x 1024 outputs of K = 2048:  128: 23.3 us, in two parts 19.7; 64: 12.1, in two parts 17.4
//   bf16,   256 x 1024 outputs of K = 16384: 128: 152.6 us whole, 30.9 in sixteen parts; 64: 66.1 whole, 24.4 in four
// f32 steps are bound by their matrix instructions, a sixteenth of bf16's rate; operands staged through registers cost
// about twice the direct loads' step.
struct GemmPlan { int F, parts, kper; };
GemmPlan gemm_plan(int es, long M, long N, long K, bool dma) {
    struct Cost { int F; double fixed, busy, lone; };
    static const Cost bf16_dma[3] = {{8, 11.0, 1.5, 1.5}, {4, 3.4, 0.45, 0.60}, {2, 1.7, 0.17, 0.25}};
    static const Cost bf16_reg[2] = {{4, 3.4, 0.80, 1.20}, {2, 1.7, 0.34, 0.50}};
    static const Cost f32[2] = {{4, 4.0, 1.90, 2.0}, {2, 1.8, 0.50, 0.55}};
    const Cost* costs = es == 4 ? f32 : dma ? bf16_dma : bf16_reg;
    const int n = es == 2 && dma ? 3 : 2;
    const long bk = 128 / es, steps = K > 0 ? (K + bk - 1) / bk : 1;
    GemmPlan best = {2, 1, (int)steps};
    double least = 1e30;
    for (int i = 0; i < n; ++i) {
        const long t = 32 * costs[i].F, tiles = ((M + t - 1) / t) * ((N + t - 1) / t);
        for (long want = 1; want <= 64 && want <= steps; want *= 2) {
            const long kper = (steps + want - 1) / want, parts = (steps + kper - 1) / kper;
            const long per_cu = (tiles * parts + 255) / 256;
            double us = per_cu <= 1 ? costs[i].fixed + kper * costs[i].lone : per_cu * (costs[i].fixed + kper * costs[i].busy);
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
long gemm_part_floats(const GemmPlan& p, long M, long N) { return p.parts > 1 ? p.parts * M * ((N + 7) & ~7L) : 0; }

template <typename T, bool AKC, bool BKC, int F, bool DMA>
int gemm_launch(const GemmArgs& a, unsigned grid, hipStream_t s) {
    static bool done[kMaxDevices] = {};
    constexpr int lds = 2 * gemm_stages(F, DMA) * GemmOperand<T, AKC, F>::BYTES;
    LDM_TRY(allow_dynamic_lds((const void*)&gemm_kernel<T, AKC, BKC, F, DMA>, lds, done));
    gemm_kernel<T, AKC, BKC, F, DMA><<<grid, 256, lds, s>>>(a);
    LDM_HIP(hipGetLastError());
    return LDM_OK;
}

template <typename T, bool AKC, bool BKC>
int gemm(GemmArgs a, float* ws, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return LDM_OK;
    constexpr long V = 16 / sizeof(T);
    auto aligned = [&](const void* p, long ld, long len) {
        return (size_t)p % 16 == 0 && ld % V == 0 && len % V == 0 && ld <= (1L << 21);
    };
    const bool dma = aligned(a.A, a.lda, AKC ? a.K : a.M) && aligned(a.B, a.ldb, BKC ? a.K : a.N);
    LDM_REQUIRE(a.lda <= (1L << 21) && a.ldb <= (1L << 21), "operand rows are more than 2^21 elements apart");
    const GemmPlan p = gemm_plan(sizeof(T), a.M, a.N, a.K, dma);
    LDM_REQUIRE(p.parts == 1 || ws, "this product needs a workspace");
    const long t = 32 * p.F, tiles = ((a.M + t - 1) / t) * ((a.N + t - 1) / t) * p.parts;
    LDM_REQUIRE(tiles < (1L << 31), "more output tiles than one launch holds");
    a.kper = p.kper;
    a.part = p.parts > 1 ? ws : nullptr;
    if (!dma && p.F == 2) LDM_TRY((gemm_launch<T, AKC, BKC, 2, false>(a, (unsigned)tiles, s)));
    else if (!dma) LDM_TRY((gemm_launch<T, AKC, BKC, 4, false>(a, (unsigned)tiles, s)));
    else if (p.F == 2) LDM_TRY((gemm_launch<T, AKC, BKC, 2, true>(a, (unsigned)tiles, s)));
    else if (p.F == 4) LDM_TRY((gemm_launch<T, AKC, BKC, 4, true>(a, (unsigned)tiles, s)));
    else if constexpr (sizeof(T) == 2) LDM_TRY((gemm_launch<T, AKC, BKC, 8, true>(a, (unsigned)tiles, s)));
    if (p.parts > 1) {
        const long n = a.M * ((a.N + 7) / 8);
        gemm_join_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, p.parts);
        LDM_HIP(hipGetLastError());
    }
    return LDM_OK;
}
template <typename T>
int gemm_by_order(const GemmArgs& a, bool akc, bool bkc, float* ws, hipStream_t s) {
    return akc ? (bkc ? gemm<T, true, true>(a, ws, s) : gemm<T, true, false>(a, ws, s)) : gemm<T, false, false>(a, ws, s);
}

// threads per row of the dz kernel, workgroups along the rows (at least four rows a thread where there are that many) and
// along the columns
struct DzShape { int ct; long groups, blocks; };
DzShape dz_shape(int es, long M, long N) {
    const long nvec = (N * es + 15) / 16;
    DzShape d;
    d.ct = 1;
    while (d.ct < 256 && d.ct < nvec) d.ct *= 2;
    d.blocks = (nvec + d.ct - 1) / d.ct;
    const long rows = (M + 256 / d.ct - 1) / (256 / d.ct);
    d.groups = (rows + 3) / 4;
    const long most = d.blocks < 1024 ? 1024 / d.blocks : 1;
    if (d.groups > most) d.groups = most;
    return d;
}

}  // namespace

int launch_gemm(int dtype, const GemmArgs& a, bool akc, bool bkc, float* ws, hipStream_t s) {
    return dtype == LDM_BF16 ? gemm_by_order<__bf16>(a, akc, bkc, ws, s) : gemm_by_order<float>(a, akc, bkc, ws, s);
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
                     long N, int act, hipStream_t s) {
    const DzShape d = dz_shape(sizeof(T), M, N);
    LDM_REQUIRE(d.blocks <= 65535, "too many columns for one launch");
    if (M > 0 && (act != LIN_NONE || db)) {
        linear_dz_kernel<T><<<dim3((unsigned)d.groups, (unsigned)d.blocks), 256, 0, s>>>(
            (const T*)dy, lddy, (const T*)pre, ldp, (T*)dz, lddz, db ? ws : nullptr, M, N, act, d.ct);
        LDM_HIP(hipGetLastError());
    }
    if (!db) return LDM_OK;
    return launch_colsum(ws, (int)d.groups, (int)N, 1, db, nullptr, s);
}
int launch_linear_dz(int dtype, const void* dy, long lddy, const void* pre, long ldp, void* dz, long lddz, float* db, float* ws,
                     long M, long N, int act, hipStream_t s) {
    return dtype == LDM_BF16 ? dz_launch<__bf16>(dy, lddy, pre, ldp, dz, lddz, db, ws, M, N, act, s)
                             : dz_launch<float>(dy, lddy, pre, ldp, dz, lddz, db, ws, M, N, act, s);
}

}  // namespace ldm
