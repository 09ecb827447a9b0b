// Rotary positions over up to four axes (time, height, width, ...): the pair j of a head's vector belongs to axis s(j) and
// turns by the angle t = pos_s * f_j:   (a, b) -> (a cos t - b sin t, a sin t + b cos t);   backward: by -t.
// Elements behind the rotated pairs pass through.  Queries and keys, which share positions, go through one launch.
// Bound by HBM: one read and one write per element.  A thread holds the angles of one 16-byte vector's pairs in registers
// and applies them to a group of heads of one token, so the trigonometry is paid once per group.
// Angles: the product of a position (below 2^29) and an f32 frequency is exact in f64; it is reduced to a fraction of a
// turn in f64 and only that fraction goes through f32 sine and cosine, so far positions lose nothing.
#include "blocks.h"

namespace ldm {

namespace {

template <typename T> struct RoVec;
template <> struct RoVec<float> {
    static constexpr int N = 4;
    typedef float V __attribute__((ext_vector_type(4), aligned(4)));
    typedef float F __attribute__((ext_vector_type(4)));
};
template <> struct RoVec<__bf16> {
    static constexpr int N = 8;
    typedef __bf16 V __attribute__((ext_vector_type(8), aligned(2)));
    typedef float F __attribute__((ext_vector_type(8)));
};

// n (<= N) elements at p; zero behind them
template <typename T>
__device__ __forceinline__ void ro_load(const T* p, int n, float* o) {
    constexpr int N = RoVec<T>::N;
    if (n >= N) {
        const typename RoVec<T>::F v = __builtin_convertvector(*(const typename RoVec<T>::V*)p, typename RoVec<T>::F);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = v[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = e < n ? (float)p[e] : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void ro_store(T* p, int n, const float* o) {
    constexpr int N = RoVec<T>::N;
    if (n >= N) {
        typename RoVec<T>::F v;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = o[e];
        *(typename RoVec<T>::V*)p = __builtin_convertvector(v, typename RoVec<T>::V);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < n) p[e] = (T)o[e];
    }
}

template <typename T, bool INTER>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    constexpr int N = RoVec<T>::N;
    const int local = threadIdx.x / a.nchunk, chunk = threadIdx.x - local * a.nchunk;
    const long token = (long)blockIdx.x * a.tpb + local;
    if (local >= a.tpb || token >= a.tokens) return;
    const unsigned b = (unsigned)token / (unsigned)a.N, n = (unsigned)token - b * (unsigned)a.N;

    // the chunk's two vectors: element offsets and counts
    int e0, e1, n0, n1;
    float cs[N], sn[N];
    const bool rot = chunk < a.nrot;
    if (rot) {
        const int j0 = chunk * N, np = a.P - j0 < N ? a.P - j0 : N;
        if constexpr (INTER) {
            e0 = 2 * j0;
            n0 = 2 * np < N ? 2 * np : N;
            e1 = e0 + N;
            n1 = 2 * np - n0;
        } else {
            e0 = j0;
            e1 = a.P + j0;
            n0 = n1 = np;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = j0 + i < a.P ? j0 + i : a.P - 1;
            int ax = 0;
#pragma unroll
            for (int k = 0; k < 3; ++k) ax += j >= a.sec_end[k];
            const long po = (long)b * a.pos_sb + (long)ax * a.pos_sa + (long)n * a.pos_sn;
            const double p = a.pos_dtype == 0 ? (double)((const int*)a.pos)[po]
                             : a.pos_dtype == 1 ? (double)((const long*)a.pos)[po] : (double)((const float*)a.pos)[po];
            const double turns = p * (double)a.inv_freq[j] * 0.15915494309189533577;
            const float f = (float)(turns - rint(turns));
            sincospif(2.0f * f, &sn[i], &cs[i]);
            if (a.inverse) sn[i] = -sn[i];
        }
    } else {
        const int c0 = 2 * a.P + (chunk - a.nrot) * 2 * N, np = a.D - c0;
        e0 = c0;
        e1 = c0 + N;
        n0 = np < N ? np : N;
        n1 = np - n0 < N ? np - n0 : N;
    }
    int h = blockIdx.y * a.hpg;
    const int hend = h + a.hpg < a.H[0] + a.H[1] ? h + a.hpg : a.H[0] + a.H[1];
    for (; h < hend; ++h) {
        const int w = h >= a.H[0];
        const int hh = w ? h - a.H[0] : h;
        const T* src = (const T*)a.in[w] + ((long)b * a.isb[w] + (long)n * a.isn[w] + (long)hh * a.ish[w]);
        T* dst = (T*)a.out[w] + ((long)b * a.osb[w] + (long)n * a.osn[w] + (long)hh * a.osh[w]);
        float u[N], v[N];
        ro_load<T>(src + e0, n0, u);
        ro_load<T>(src + e1, n1, v);
        if (rot) {
            if constexpr (INTER) {
#pragma unroll
                for (int i = 0; i < N / 2; ++i) {
                    const float x0 = u[2 * i], y0 = u[2 * i + 1], x1 = v[2 * i], y1 = v[2 * i + 1];
                    u[2 * i] = x0 * cs[i] - y0 * sn[i];
                    u[2 * i + 1] = x0 * sn[i] + y0 * cs[i];
                    v[2 * i] = x1 * cs[N / 2 + i] - y1 * sn[N / 2 + i];
                    v[2 * i + 1] = x1 * sn[N / 2 + i] + y1 * cs[N / 2 + i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float x = u[i], y = v[i];
                    u[i] = x * cs[i] - y * sn[i];
                    v[i] = x * sn[i] + y * cs[i];
                }
            }
        }
        ro_store<T>(dst + e0, n0, u);
        ro_store<T>(dst + e1, n1, v);
    }
}

}  // namespace

int launch_rope(int dtype, int interleaved, RopeArgs a, hipStream_t s) {
    const int N = dtype == LDM_BF16 ? 8 : 4;
    if (a.tokens == 0) return LDM_OK;
    a.nrot = (a.P + N - 1) / N;
    a.nchunk = a.nrot + (a.D - 2 * a.P + 2 * N - 1) / (2 * N);
    a.tpb = 256 / a.nchunk;
    const int heads = a.H[0] + a.H[1];
    a.hpg = heads < 8 ? heads : 8;
    const dim3 grid((unsigned)((a.tokens + a.tpb - 1) / a.tpb), (unsigned)((heads + a.hpg - 1) / a.hpg));
    if (dtype == LDM_BF16) {
        if (interleaved) rope_kernel<__bf16, true><<<grid, 256, 0, s>>>(a);
        else rope_kernel<__bf16, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (interleaved) rope_kernel<float, true><<<grid, 256, 0, s>>>(a);
        else rope_kernel<float, false><<<grid, 256, 0, s>>>(a);
    }
    LDM_HIP(hipGetLastError());
    return LDM_OK;
}

}  // namespace ldm
