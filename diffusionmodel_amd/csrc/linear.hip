// Linear layer with its epilogue, and its backward pass:
//   z = x W + b + res,  y = act(z);     dz = dy act'(z),  dx = dz W^T,  dW = x^T dz,  db = sum_rows dz
// All three products are C[m, n] = sum_k A(m, k) B(k, n) on one kernel family; an operand is either contiguous along the
// contraction (KC) or along its other index.
#include "blocks.h"

namespace ldm {

namespace {

typedef u32x4 u32x4_u2 __attribute__((aligned(2)));
typedef u32x4 u32x4_u4 __attribute__((aligned(4)));

__device__ __forceinline__ float lin_act(float v, int act) {
    if (act == LIN_SILU) return v / (1.0f + expf(-v));
    if (act == LIN_RELU) return v < 0.f ? 0.f : v;
    if (act == LIN_GELU) return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f));
    return v;
}
__device__ __forceinline__ float lin_dact(float z, int act) {
    if (act == LIN_SILU) {
        const float s = 1.0f / (1.0f + expf(-z));
        return s * (1.0f + z * (1.0f - s));
    }
    if (act == LIN_RELU) return z > 0.f ? 1.f : 0.f;
    if (act == LIN_GELU)
        return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * expf(-0.5f * z * z) * 0.39894228040143268f;
    return 1.f;
}

template <typename T> __device__ __forceinline__ T lin_zero() { return (T)0.f; }

// 64 x 64 outputs per workgroup, 64 bytes of the contraction per step, staged through registers with every access
// guarded: serves every size, stride and alignment.
constexpr int GT = 64, GROW = 64 + 16;      // bytes of an LDS row: 64 of data, padded against bank conflicts
template <typename T, bool AKC, bool BKC>
__global__ __launch_bounds__(256) void gemm_any_kernel(GemmArgs a) {
    constexpr int ES = sizeof(T), KB = 64 / ES;
    __shared__ __attribute__((aligned(16))) char As[GT * GROW];
    __shared__ __attribute__((aligned(16))) char Bs[GT * GROW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = lane >> 4, l15 = lane & 15;
    const unsigned nt = (unsigned)((a.N + GT - 1) / GT);
    const long m0 = (long)(blockIdx.x / nt) * GT, n0 = (long)(blockIdx.x % nt) * GT;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    f32x4 acc[2][2] = {};      // [n][m]
    for (long k0 = 0; k0 < a.K; k0 += KB) {
        __syncthreads();
        for (int i = tid; i < GT * KB; i += 256) {
            int r, k;
            if (AKC) { r = i / KB; k = i % KB; } else { k = i / GT; r = i % GT; }
            T v = lin_zero<T>();
            if (m0 + r < a.M && k0 + k < a.K)
                v = ((const T*)a.A)[AKC ? (m0 + r) * a.lda + k0 + k : (k0 + k) * a.lda + m0 + r];
            *(T*)(As + r * GROW + k * ES) = v;
        }
        for (int i = tid; i < GT * KB; i += 256) {
            int r, k;
            if (BKC) { r = i / KB; k = i % KB; } else { k = i / GT; r = i % GT; }
            T v = lin_zero<T>();
            if (n0 + r < a.N && k0 + k < a.K)
                v = ((const T*)a.B)[BKC ? (n0 + r) * a.ldb + k0 + k : (k0 + k) * a.ldb + n0 + r];
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
                    // lane group g holds k = 4 g .. 4 g + 3; product q takes element q of both operands
                    const f32x4 va = __builtin_bit_cast(f32x4, fa[i]), vb = __builtin_bit_cast(f32x4, fb[j]);
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vb[q], va[q], acc[j][i], 0, 0, 0);
                }
            }
    }
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
                if (a.bias) v += a.bias[n];
                if (a.res) v += (float)((const T*)a.res)[m * a.ldr + n];
                if (a.pre) ((T*)a.pre)[m * a.ldp + n] = (T)v;
                ((T*)a.C)[m * a.ldc + n] = (T)lin_act(v, a.act);
            }
    }
}

// dz = dy act'(pre), and the column sums of dz over this workgroup's rows (part [gridDim.x][N])
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(const T* dy, long lddy, const T* pre, long ldp, T* dz, long lddz,
                                                        float* part, long M, long N, int act) {
    const long n = (long)blockIdx.y * 256 + threadIdx.x;
    if (n >= N) return;
    float s = 0.f;
    for (long m = blockIdx.x; m < M; m += gridDim.x) {
        float v = (float)dy[m * lddy + n];
        if (act != LIN_NONE) {
            v *= lin_dact((float)pre[m * ldp + n], act);
            dz[m * lddz + n] = (T)v;
        }
        s += v;
    }
    if (part) part[blockIdx.x * N + n] = s;
}

template <typename T>
int gemm(const GemmArgs& a, bool akc, bool bkc, hipStream_t s) {
    if (a.M == 0 || a.N == 0) return LDM_OK;
    const long tiles = ((a.N + GT - 1) / GT) * ((a.M + GT - 1) / GT);
    LDM_REQUIRE(tiles < (1L << 31), "more output tiles than one launch holds");
    const unsigned grid = (unsigned)tiles;
    if (akc && bkc) gemm_any_kernel<T, true, true><<<grid, 256, 0, s>>>(a);
    else if (akc) gemm_any_kernel<T, true, false><<<grid, 256, 0, s>>>(a);
    else gemm_any_kernel<T, false, false><<<grid, 256, 0, s>>>(a);
    LDM_HIP(hipGetLastError());
    return LDM_OK;
}

long dz_groups(long M, long N) { return M < 512 ? M : 512; }

}  // namespace

int launch_gemm(int dtype, const GemmArgs& a, bool akc, bool bkc, hipStream_t s) {
    return dtype == LDM_BF16 ? gemm<__bf16>(a, akc, bkc, s) : gemm<float>(a, akc, bkc, s);
}

long linear_dz_ws_floats(long M, long N) { return dz_groups(M, N) * N; }

int launch_linear_dz(int dtype, const void* dy, long lddy, const void* pre, long ldp, void* dz, long lddz, float* db, float* ws,
                     long M, long N, int act, hipStream_t s) {
    const long G = dz_groups(M, N);
    if (M > 0 && (act != LIN_NONE || db)) {
        const dim3 grid((unsigned)G, (unsigned)((N + 255) / 256));
        if (dtype == LDM_BF16)
            linear_dz_kernel<__bf16><<<grid, 256, 0, s>>>((const __bf16*)dy, lddy, (const __bf16*)pre, ldp, (__bf16*)dz, lddz,
                                                          db ? ws : nullptr, M, N, act);
        else
            linear_dz_kernel<float><<<grid, 256, 0, s>>>((const float*)dy, lddy, (const float*)pre, ldp, (float*)dz, lddz,
                                                         db ? ws : nullptr, M, N, act);
        LDM_HIP(hipGetLastError());
    }
    if (!db) return LDM_OK;
    return launch_colsum(ws, (int)G, (int)N, 1, db, nullptr, s);
}

}  // namespace ldm
