// tgkv_group.cu -- attention of several sequences of one layer that may share
// a prefix cache: token t of sequence i attends the prefix's positions [0, P)
// and its own cache's positions [0, old_i + t].  q head h reads KV head
// h * n_kv_heads / n_heads; out = softmax(q K^T * scale) V over both parts.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "tgkv_launch.h"
#include "tgkv_ptx.cuh"

namespace tgkv {
namespace group {

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<uint16_t>(uint16_t x) { return bf16_bits_to_f32(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ uint16_t from_f<uint16_t>(float x) { return f32_to_bf16_rne(x); }

// The sequence of packed token t: the last one whose first token is at or
// before t among those with tokens.
__device__ __forceinline__ uint32_t seq_of(const TGKvGroupParams& p, uint32_t t) {
    uint32_t lo = 0, hi = p.n_seq;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (p.tok0[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The packed rows of k_new / v_new into their caches, 8 elements per thread.
template <typename T>
__global__ void __launch_bounds__(256) group_append_kernel(const __grid_constant__ TGKvGroupParams p) {
    const uint32_t kv_dim = p.n_kv_heads * p.head_dim, vec = kv_dim / 8;
    const uint64_t x = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (x >= (uint64_t)p.tok0[p.n_seq] * vec) return;
    const uint32_t t = (uint32_t)(x / vec), e = (uint32_t)(x % vec) * 8, i = seq_of(p, t);
    const T* src = reinterpret_cast<const T*>(blockIdx.y ? p.v_new : p.k_new) + (uint64_t)t * kv_dim + e;
    const TGKvRowCache c = p.table[i];
    uint16_t* dst = reinterpret_cast<uint16_t*>(c.base) +
                    ((uint64_t)blockIdx.y * c.max_seq + p.old_len[i] + (t - p.tok0[i])) * kv_dim + e;
    uint4 w;
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
        w = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
    } else {
        w = *reinterpret_cast<const uint4*>(src);
    }
    *reinterpret_cast<uint4*>(dst) = w;
}

// One warp per (token, query head): the positions one after another with the
// online softmax, HD / 32 head dims per lane.
template <typename T, int HD>
__global__ void __launch_bounds__(128) group_simple_kernel(const __grid_constant__ TGKvGroupParams p) {
    constexpr int D = HD / 32;
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= p.tok0[p.n_seq] * p.n_heads) return;
    const uint32_t t = row / p.n_heads, h = row % p.n_heads, i = seq_of(p, t);
    const uint32_t kv_dim = p.n_kv_heads * HD, col = h / (p.n_heads / p.n_kv_heads) * HD + lane * D;
    float q[D], o[D], m = -INFINITY, l = 0.f;
    const T* qp = reinterpret_cast<const T*>(p.q) + (uint64_t)row * HD + lane * D;
#pragma unroll
    for (int d = 0; d < D; ++d) { q[d] = to_f<T>(qp[d]) * p.qscale; o[d] = 0.f; }
    for (int part = 0; part < 2; ++part) {
        const uint32_t n = part ? p.old_len[i] + (t - p.tok0[i]) + 1 : p.prefix_len;
        if (n == 0) continue;
        const TGKvRowCache c = p.table[part ? i : p.n_seq];
        const uint16_t* k = reinterpret_cast<const uint16_t*>(c.base) + col;
        const uint16_t* v = k + (uint64_t)c.max_seq * kv_dim;
        for (uint32_t j = 0; j < n; ++j) {
            float s = 0.f;
#pragma unroll
            for (int d = 0; d < D; ++d) s += q[d] * bf16_bits_to_f32(k[(uint64_t)j * kv_dim + d]);
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
            const float m2 = fmaxf(m, s), a = exp2f(m - m2), e = exp2f(s - m2);
            l = l * a + e;
#pragma unroll
            for (int d = 0; d < D; ++d) o[d] = o[d] * a + e * bf16_bits_to_f32(v[(uint64_t)j * kv_dim + d]);
            m = m2;
        }
    }
    T* op = reinterpret_cast<T*>(p.out) + (uint64_t)row * HD + lane * D;
#pragma unroll
    for (int d = 0; d < D; ++d) op[d] = from_f<T>(o[d] / l);
}

template <typename T, int HD>
int launch(const TGKvGroupParams* p, cudaStream_t st) {
    const uint32_t total = p->tok0[p->n_seq];
    if (p->k_new) {
        const uint64_t n = (uint64_t)total * (p->n_kv_heads * HD / 8);
        group_append_kernel<T><<<dim3((unsigned)((n + 255) / 256), 2), 256, 0, st>>>(*p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int)e;
    }
    group_simple_kernel<T, HD><<<(total * p->n_heads + 3) / 4, 128, 0, st>>>(*p);
    return (int)cudaGetLastError();
}

}  // namespace group
}  // namespace tgkv

extern "C" int tgkv_launch_group(const TGKvGroupParams* p, int act, void* stream) {
    using namespace tgkv::group;
    cudaStream_t st = (cudaStream_t)stream;
    if (p->head_dim == 128) return act ? launch<uint16_t, 128>(p, st) : launch<float, 128>(p, st);
    if (p->head_dim == 64) return act ? launch<uint16_t, 64>(p, st) : launch<float, 64>(p, st);
    return (int)cudaErrorInvalidValue;
}
