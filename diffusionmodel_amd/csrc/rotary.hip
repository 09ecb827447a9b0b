// Rotary positions over up to four axes (time, height, width, ...): the pair j of a head's vector belongs to axis s(j) and
// turns by the angle t = pos_s * f_j:   (a, b) -> (a cos t - b sin t, a sin t + b cos t);   backward: by -t.
// Elements behind the rotated pairs pass through.  Queries and keys, which share positions, go through one launch.
// Bound by HBM: one read and one write per element.  A thread holds the angles of one 16-byte vector's pairs in registers
// and applies them to a group of heads of one token, so the trigonometry is paid once per group.
// 2 x 8192 tokens, 20 heads of 128 f32: 69 us = 4.9 TB/s (a large copy: 5.0); 64 x 256 tokens, 8 heads of 64 bf16 out of a
// fused projection: 9.1 us, of which the first loads, the angles and the launch are about half.
// Angles: the product of a position (below 2^29) and an f32 frequency is exact in f64; it is reduced to a fraction of a
// turn in f64 and only that fraction goes through f32 sine and cosine, so far positions lose nothing.
#include "blocks.h"
#include "vec.h"

namespace ldm {

namespace {

// sine and cosine of a fraction of a turn: the nearest quarter is taken off in f64, the rest (at most an eighth, so that
// its rounding to f32 is 2^-28 of a turn) goes through the Taylor series up to x^9 and x^10, which |x| <= pi / 4 leaves
// exact to 2e-9
__device__ __forceinline__ void turn_sincos(double turns, float& sn, float& cs) {
    const double q4 = turns * 4.0, q = rint(q4);
    const float x = (float)(q4 - q) * 1.57079632679489662f;
    // the quarter modulo four: a double of this size holds it exactly
    const int k = (int)(q - 4.0 * rint(q * 0.25));
    const float y = x * x;
    float s = __builtin_fmaf(y, 2.7557319224e-6f, -1.9841269841e-4f);
    s = __builtin_fmaf(y, s, 8.3333333333e-3f);
    s = __builtin_fmaf(y, s, -1.6666666667e-1f);
    s = __builtin_fmaf(x * y, s, x);
    float c = __builtin_fmaf(y, -2.7557319224e-7f, 2.4801587302e-5f);
    c = __builtin_fmaf(y, c, -1.3888888889e-3f);
    c = __builtin_fmaf(y, c, 4.1666666667e-2f);
    c = __builtin_fmaf(y, c, -0.5f);
    c = __builtin_fmaf(y, c, 1.0f);
    const float a = (k & 1) ? c : s, b = (k & 1) ? s : c;
    sn = (k & 2) ? -a : a;
    cs = ((k + 1) & 2) ? -b : b;
}

constexpr int kRopeMost = 320;        // threads of a workgroup whose head takes one chunk more than 256

template <typename T, bool INTER>
__global__ __launch_bounds__(kRopeMost) void rope_kernel(RopeArgs a) {
    constexpr int N = RowVec<T>::N;
    const int local = threadIdx.x / a.nchunk, chunk = threadIdx.x - local * a.nchunk;
    // the head groups of the same tokens follow each other, so that a token's heads are read at about the same time
    const unsigned blk = blockIdx.x / a.groups, grp = blockIdx.x - blk * a.groups;
    const long token = (long)blk * a.tpb + local;
    if (local >= a.tpb || token >= a.tokens) return;
    const unsigned b = (unsigned)token / (unsigned)a.N, n = (unsigned)token - b * (unsigned)a.N;

    // the chunk's two vectors: element offsets and counts
    int e0, e1, n0, n1;
    const bool rot = chunk < a.nrot;
    const int j0 = chunk * N;
    // (pairs side by side: two vectors that stand half a head apart, so that the lanes of each access are neighbours)
    if (rot && !INTER) {
        e0 = j0;
        e1 = a.P + j0;
        n0 = n1 = a.P - j0;
    } else {
        const int first = rot ? 0 : 2 * a.P, last = rot ? 2 * a.P : a.D, half = rot ? a.nrot : a.nchunk - a.nrot;
        e0 = first + (rot ? chunk : chunk - a.nrot) * N;
        e1 = e0 + half * N;
        n0 = last - e0;
        n1 = last - e1;
    }
    // four heads at a time: the next four are on their way while these are turned, the first while the angles are taken
    const int heads = a.H[0] + a.H[1], h0 = grp * a.hpg, hend = h0 + a.hpg < heads ? h0 + a.hpg : heads;
    typename RowVec<T>::R nu[4], nv[4];
    auto fetch = [&](int h) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (h + d >= hend) continue;
            const int w = h + d >= a.H[0], hh = w ? h + d - a.H[0] : h + d;
            const T* src = (const T*)a.in[w] + ((long)b * a.isb[w] + (long)n * a.isn[w] + (long)hh * a.ish[w]);
            nu[d] = row_load<T>(src + e0, n0);
            nv[d] = row_load<T>(src + e1, n1);
        }
    };
    fetch(h0);
    float cs[N], sn[N];
    if (rot) {
        // the token's position on each axis and the pairs' frequencies, every load before the first use
        double pos[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const long po = (long)b * a.pos_sb + (long)(k < a.axes ? k : 0) * a.pos_sa + (long)n * a.pos_sn;
            pos[k] = a.pos_dtype == 0 ? (double)((const int*)a.pos)[po]
                     : a.pos_dtype == 1 ? (double)((const long*)a.pos)[po] : (double)((const float*)a.pos)[po];
        }
        float f[N];
        // the pairs' numbers: j0 .. j0 + N - 1, or half of them from each vector
        const int j1 = INTER ? e0 / 2 : j0, j2 = INTER ? e1 / 2 - N / 2 : j0;
#pragma unroll
        for (int i = 0; i < N; i += INTER ? N / 2 : 4) {
            const int j = (i < N / 2 ? j1 : j2) + i, most = INTER ? N / 2 : 4;
            float t[4];
            row_floats<float>(row_load<float>(a.inv_freq + j, a.P - j < most ? a.P - j : most), t);
#pragma unroll
            for (int e = 0; e < most; ++e) f[i + e] = t[e];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (i < N / 2 ? j1 : j2) + i;
            const double p = j < a.sec_end[0] ? pos[0] : j < a.sec_end[1] ? pos[1] : j < a.sec_end[2] ? pos[2] : pos[3];
            const double turns = p * (double)f[i] * 0.15915494309189533577;
            turn_sincos(a.inverse ? -turns : turns, sn[i], cs[i]);
        }
    }
    for (int h = h0; h < hend; h += 4) {
        typename RowVec<T>::R lu[4], lv[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            lu[d] = nu[d];
            lv[d] = nv[d];
        }
        fetch(h + 4);
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (h + d >= hend) continue;
            const int w = h + d >= a.H[0], hh = w ? h + d - a.H[0] : h + d;
            T* dst = (T*)a.out[w] + ((long)b * a.osb[w] + (long)n * a.osn[w] + (long)hh * a.osh[w]);
            float u[N], v[N];
            row_floats<T>(lu[d], u);
            row_floats<T>(lv[d], v);
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
            row_store<T>(dst + e0, n0, u, a.through);
            row_store<T>(dst + e1, n1, v, a.through);
        }
    }
}

}  // namespace

int launch_rope(int dtype, int interleaved, RopeArgs a, hipStream_t s) {
    const int N = dtype == LDM_BF16 ? 8 : 4;
    if (a.tokens == 0) return LDM_OK;
    a.nrot = interleaved ? ((2 * a.P + N - 1) / N + 1) / 2 : (a.P + N - 1) / N;      // two vectors a thread
    a.nchunk = a.nrot + (a.D - 2 * a.P + 2 * N - 1) / (2 * N);
    // a head of 2048 f32 elements whose rotated pairs end inside a vector has 257 chunks
    const int threads = a.nchunk > 256 ? kRopeMost : 256;
    LDM_REQUIRE(a.nchunk <= threads, "a head is longer than a workgroup");
    a.tpb = threads / a.nchunk;
    // a group of heads per workgroup, all of them where the tokens alone give eight workgroups per CU: the angles are taken
    // once for a group.  2 x 8192 tokens, 20 heads of 128 in f32: 69.6 us in two groups of ten, 72.8 in one, 70.6 in four, 93
    // with a workgroup per head; 64 x 256 tokens, 8 heads of 64 in bf16: 9.1 in four groups, 9.5 in one, 12.5 per head; one
    // token, 8 heads of 64: 4.7 in four, 7.6 in one
    const int heads = a.H[0] + a.H[1], es = dtype == LDM_BF16 ? 2 : 4;
    const long blocks = (a.tokens + a.tpb - 1) / a.tpb;
    long groups = 2048 / blocks;
    groups = groups < 1 ? 1 : groups > (heads + 1) / 2 ? (heads + 1) / 2 : groups;
    a.hpg = (int)((heads + groups - 1) / groups);
    a.groups = (unsigned)((heads + a.hpg - 1) / a.hpg);
    // written through where each access of the lanes covers half lines at least (the second access fills them)
    a.through = a.tokens * heads * a.D * es <= kThroughBytes && (interleaved ? 2 : 1) * a.P * es % 64 == 0 && a.D * es % 64 == 0;
    for (int w = 0; w < 2 && a.H[w]; ++w)
        a.through = a.through && ((size_t)a.out[w] | (size_t)(a.osb[w] * es) | (size_t)(a.osn[w] * es) | (size_t)(a.osh[w] * es)) % 64 == 0;
    LDM_REQUIRE(blocks * a.groups * threads < (1L << 32), "too many tokens and heads for one launch");
    const unsigned grid = (unsigned)(blocks * a.groups);
    if (dtype == LDM_BF16) {
        if (interleaved) rope_kernel<__bf16, true><<<grid, threads, 0, s>>>(a);
        else rope_kernel<__bf16, false><<<grid, threads, 0, s>>>(a);
    } else {
        if (interleaved) rope_kernel<float, true><<<grid, threads, 0, s>>>(a);
        else rope_kernel<float, false><<<grid, threads, 0, s>>>(a);
    }
    LDM_HIP(hipGetLastError());
    return LDM_OK;
}

}  // namespace ldm
