// Device helpers shared by the token-sequence kernels (norm_rows.hip, causal_conv.hip, scan.hip).
#pragma once
#include "bf16_common.hpp"

namespace rst {

// A launch has fewer than 2^32 threads along x.  More blocks than that go into rows of 2^31 / THREADS blocks along y; the last
// row then has blocks past the end, which a kernel sends home.
template <int THREADS> static dim3 grid_of(int64_t blocks) {
    constexpr int64_t ROW = (1ll << 31) / THREADS;
    return blocks <= ROW ? dim3((unsigned)blocks) : dim3((unsigned)ROW, (unsigned)cdiv(blocks, ROW));
}
template <int THREADS> __device__ __forceinline__ uint32_t block_index() {
    return blockIdx.y * (uint32_t)((1ll << 31) / THREADS) + blockIdx.x;
}

// Values per 16 bytes, and conversions of the two storage types.  All arithmetic is fp32; a bf16 result is rounded
// once, to nearest even, when it is stored.
template <typename T> struct Store;
template <> struct Store<float> {
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Store<bf16_t> {
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float get(bf16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ bf16_t put(float v) { return to_bf16_bits(v); }
};

// K consecutive values as they lie in memory.  Rows of an odd length start anywhere, so nothing is assumed about
// the address beyond that of one value: gfx950 takes wide loads and stores of global memory at any address (the
// compiler forms them from the copies below).
template <typename T, int K> struct Raw {
    uint32_t w[(K * (int)sizeof(T) + 3) / 4];
    __device__ __forceinline__ void load(const T* p) { w[0] = 0; __builtin_memcpy(w, p, K * sizeof(T)); }
    __device__ __forceinline__ void store(T* p) const { __builtin_memcpy(p, w, K * sizeof(T)); }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return (i & 1) ? bf_hi(w[i >> 1]) : bf_lo(w[i >> 1]);
    }
    __device__ __forceinline__ void unpack(float (&v)[K]) const {
#pragma unroll
        for (int i = 0; i < K; ++i) v[i] = get(i);
    }
    __device__ __forceinline__ void pack(const float (&v)[K]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < K; ++i) w[i] = __float_as_uint(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < (K + 1) / 2; ++i) w[i] = pack_bf16(v[2 * i], 2 * i + 1 < K ? v[2 * i + 1] : 0.f);
        }
    }
};

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp_fast(float v) { return __builtin_amdgcn_exp2f(v * LOG2E); }
__device__ __forceinline__ float rcp_fast(float v) { return __builtin_amdgcn_rcpf(v); }     // 1 ulp
// 1 / (1 + e^-v): e^-v = inf for a very negative v gives 0, as it should
__device__ __forceinline__ float sigmoid(float v) { return rcp_fast(1.0f + exp_fast(-v)); }

}  // namespace rst
