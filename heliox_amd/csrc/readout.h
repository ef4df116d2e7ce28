// Readout operators over a network's captured outputs: linear attention with a decay for
// each head (readout_attention.hip), a gated recurrence (readout_recurrence.hip), layer norm
// (readout_norm.hip), the loss against a teacher's top logits (readout_distill.hip), log
// probabilities of given tokens (readout_logprob.hip), the drawing of an answer
// (readout_sample.hip) and the step of the parameters (readout_adamw.hip).  readout.cpp holds
// the C entry points and their checks; the kernels take the checked arguments.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>

#include "heliox.h"

namespace hx {

constexpr int kAttnMaxDim = 256;
constexpr int64_t kDistillMaxVocab = 1 << 20;
constexpr int64_t kDistillMaxTop = 2048;
constexpr int64_t kLogprobMaxTop = 256;

// Each launches on the arguments' stream; the sizes are checked and not zero.
size_t attention_workspace(const hx_attention_args& A, bool grad);
hipError_t attention_forward(const hx_attention_args& A);
hipError_t attention_backward(const hx_attention_args& A);
hipError_t attention_step(const hx_attention_args& A);
hipError_t distill_launch(const hx_distill_args& A);
hipError_t sample_launch(const hx_sample_args& A);
size_t norm_workspace(const hx_norm_args& A);
hipError_t norm_forward(const hx_norm_args& A);
hipError_t norm_backward(const hx_norm_args& A);
size_t recurrence_workspace(const hx_recurrence_args& A, bool grad);
hipError_t recurrence_forward(const hx_recurrence_args& A);
hipError_t recurrence_backward(const hx_recurrence_args& A);
hipError_t recurrence_step(const hx_recurrence_args& A);
size_t logprob_workspace(const hx_logprob_args& A);
hipError_t logprob_launch(const hx_logprob_args& A);
hipError_t logprob_gradient(const hx_logprob_args& A);
hipError_t adamw_launch(const hx_adamw_args& A);

template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32<__hip_bfloat16>(__hip_bfloat16 x) { return __bfloat162float(x); }

template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half(x); }
template <> __device__ __forceinline__ __hip_bfloat16 from_f32<__hip_bfloat16>(float x) {
    return __float2bfloat16(x);
}

// 16 bytes of a row of logits; pieces start at any element.
template <class T> struct PieceOf;
template <> struct PieceOf<float> { typedef float Vec __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct PieceOf<__half> { typedef _Float16 Vec __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct PieceOf<__hip_bfloat16> { typedef __bf16 Vec __attribute__((ext_vector_type(8), aligned(2))); };

// x reduced over the workgroup's waves, by way of sh (one for each wave); every thread gets the result.
template <int kThreads, class W, class V, class F>
__device__ __forceinline__ V block_reduce(V x, W* sh, F op) {
    for (int m = 32; m > 0; m >>= 1) x = op(x, __shfl_xor(x, m));
    __syncthreads();
    if (threadIdx.x % 64 == 0) sh[threadIdx.x / 64] = x;
    __syncthreads();
    x = static_cast<V>(sh[threadIdx.x % (kThreads / 64)]);
    for (int m = kThreads / 128; m > 0; m >>= 1) x = op(x, __shfl_xor(x, m));
    return x;
}

// Calls f with a value of the element type that `type` names.
template <class F>
auto with_type(int64_t type, F&& f) {
    switch (type) {
        case HX_F16: return f(__half{});
        case HX_BF16: return f(__hip_bfloat16{});
        default: return f(float{});
    }
}

}  // namespace hx
