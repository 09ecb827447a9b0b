// 16-byte vectors of a row at element alignment, and sums over a row's lanes (device code of the transformer blocks).
#pragma once
#include <hip/hip_runtime.h>

namespace ldm {

// Whether an output of `bytes` is written through: what the caches hold of it at the end of a launch is at most some 32 MB,
// a few us; against large outputs that is nothing and the detour costs (65536 x 1024 bf16 behind a product: 1 % slower,
// 16384 x 1024 with its value before the activation 6 % faster).
constexpr long kThroughBytes = 96L << 20;

// N elements of T as one 16-byte access.  The rows of a slice are element aligned only; this target's global memory serves
// such accesses at any address that the element allows.
template <typename T> struct RowVec;
template <> struct RowVec<float> {
    static constexpr int N = 4;
    typedef float V __attribute__((ext_vector_type(4), aligned(4)));
    typedef float F __attribute__((ext_vector_type(4)));
    typedef float R __attribute__((ext_vector_type(4)));            // the same, in a register
};
template <> struct RowVec<__bf16> {
    static constexpr int N = 8;
    typedef __bf16 V __attribute__((ext_vector_type(8), aligned(2)));
    typedef float F __attribute__((ext_vector_type(8)));
    typedef __bf16 R __attribute__((ext_vector_type(8)));
};

// the first n elements at p, zeros for the rest; n may be zero or less, or more than all
template <typename T>
__device__ __forceinline__ typename RowVec<T>::R row_load(const T* p, int n) {
    constexpr int N = RowVec<T>::N;
    typename RowVec<T>::R v = {};
    if (n >= N) {
        v = *(const typename RowVec<T>::V*)p;
    } else if (n > 0) {
        asm volatile("" ::: "memory");          // a branch of its own: lanes behind the end would walk through it as well
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
            if (e < n) v[e] = p[e];
    }
    return v;
}
// 16 bytes, written through: nothing dirty is left in this XCD's L2 for the end of the launch, which would have to write it
// back before the next launch starts.  Only for stores that cover whole lines at once: partial ones go to memory one by one
// (20011 rows of 1031 f32: 67 us against 34 written back).  The s_nop keeps the data registers until the store has read
// them: the compiler does not know the instruction.
template <typename R> __device__ __forceinline__ void store_through(void* p, const R& v) {
    asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" ::"v"(p), "v"(v) : "memory");
}
template <typename T>
__device__ __forceinline__ void row_store(T* p, int n, const float* o, bool through = false) {
    constexpr int N = RowVec<T>::N;
    typename RowVec<T>::F f;
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = o[e];
    const typename RowVec<T>::R v = __builtin_convertvector(f, typename RowVec<T>::R);
    if (n >= N) {
        if (through) store_through(p, v);
        else *(typename RowVec<T>::V*)p = v;
    } else if (n > 0) {
        asm volatile("" ::: "memory");
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
            if (e < n) p[e] = v[e];
    }
}
template <typename T>
__device__ __forceinline__ void row_floats(const typename RowVec<T>::R& v, float* o) {
    const typename RowVec<T>::F f = __builtin_convertvector(v, typename RowVec<T>::F);
#pragma unroll
    for (int e = 0; e < RowVec<T>::N; ++e) o[e] = f[e];
}

// a + the value of the lane that DPP control C names (all lanes take part)
template <int C> __device__ __forceinline__ float lane_add(float a) {
    return a + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, a), C, 0xf, 0xf, true));
}
// sum over groups of L consecutive lanes (L = 8, 16, 32, 64), the same bits in every lane of the group: in the VALU (quad
// permutations, mirrors, row swaps), where a shuffle through LDS would cost its latency at each step
template <int L> __device__ __forceinline__ float lanes_sum(float a) {
    a = lane_add<0xB1>(a);           // lane ^ 1
    a = lane_add<0x4E>(a);           // lane ^ 2
    a = lane_add<0x141>(a);          // mirror within 8
    if constexpr (L >= 16) a = lane_add<0x140>(a);       // mirror within 16
    if constexpr (L >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, a), false, false);
        const unsigned s0 = s[0], s1 = s[1];
        a = __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
    }
    if constexpr (L >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, a), __builtin_bit_cast(unsigned, a), false, false);
        const unsigned s0 = s[0], s1 = s[1];
        a = __builtin_bit_cast(float, s0) + __builtin_bit_cast(float, s1);
    }
    return a;
}

}  // namespace ldm
