// The loss against a teacher's top logits, and its gradient by the student's, one workgroup
// per row.
#include "readout.h"

namespace hx {
namespace {

constexpr int kThreads = 256;

struct Pair {          // running maximum and the sum of e^{x - max}
    float m, s;
};

__device__ __forceinline__ float exp_diff(float a, float b) { return a == b ? 1.f : expf(a - b); }

__device__ __forceinline__ Pair join(Pair a, Pair b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s};
    return {m, a.s * exp_diff(a.m, m) + b.s * exp_diff(b.m, m)};
}

template <class F>
__device__ __forceinline__ float block_sum(float x, float* sh, F op) {
    for (int m = 32; m > 0; m >>= 1) x = op(x, __shfl_xor(x, m));
    __syncthreads();
    if (threadIdx.x % 64 == 0) sh[threadIdx.x / 64] = x;
    __syncthreads();
    x = sh[0];
    for (int w = 1; w < kThreads / 64; ++w) x = op(x, sh[w]);
    return x;
}

template <class I>
__device__ __forceinline__ int entry(const void* index, long long at, int vocab) {
    const I j = static_cast<const I*>(index)[at];
    return j >= 0 && j < vocab ? static_cast<int>(j) : -1;
}

// LDS: places and teacher's shares of the row's entries, the student's logits there, and one
// bit for each place of the vocabulary that holds an entry.
template <class T, class U, class I>
__global__ void __launch_bounds__(kThreads) k_distill(hx_distill_args A) {
    extern __shared__ int lds[];
    __shared__ float red[kThreads / 64];
    const int top = static_cast<int>(A.top), vocab = static_cast<int>(A.vocab);
    int* place = lds;
    float* share = reinterpret_cast<float*>(lds + top);
    float* logq = share + top;
    unsigned* member = reinterpret_cast<unsigned*>(logq + top);
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(A.logits) + row * A.logits_stride;
    const U* t = static_cast<const U*>(A.teacher) + row * A.teacher_stride;
    const float cold = 1.f / static_cast<float>(A.temperature), tau = static_cast<float>(A.temperature);
    const bool rest = A.teacher_lse != nullptr;
    auto add = [](float a, float b) { return a + b; };
    auto most = [](float a, float b) { return fmaxf(a, b); };

    for (int w = threadIdx.x; w < (vocab + 31) / 32; w += kThreads) member[w] = 0;
    __syncthreads();
    float tmax = -INFINITY, some = 0.f;
    for (int k = threadIdx.x; k < top; k += kThreads) {
        const int j = entry<I>(A.index, row * A.index_stride + k, vocab);
        place[k] = j;
        share[k] = j >= 0 ? to_f32(t[k]) * cold : -INFINITY;
        logq[k] = j >= 0 ? to_f32(x[j]) * cold : 0.f;
        if (j >= 0) {
            some = 1.f;
            tmax = fmaxf(tmax, share[k]);
            atomicOr(member + j / 32, 1u << (j % 32));
        }
    }
    some = block_sum(some, red, most);
    tmax = block_sum(tmax, red, most);

    // the student's maximum and sums: all places, and those without an entry
    Pair all{-INFINITY, 0.f};
    float others = 0.f;
    for (int j = threadIdx.x; j < vocab; j += kThreads) {
        const float v = to_f32(x[j]) * cold;
        const bool in = member[j / 32] >> (j % 32) & 1;
        const float m = v != v ? v : fmaxf(all.m, v);
        const float keep = all.m == m ? 1.f : expf(all.m - m), e = v == -INFINITY ? 0.f : exp_diff(v, m);
        all = {m, all.s * keep + e};
        others = others * keep + (in ? 0.f : e);
    }
    const float m = block_sum(all.m, red, most);
    const float scale = all.m == -INFINITY ? 0.f : exp_diff(all.m, m);
    const float z = block_sum(all.s * scale, red, add);
    others = block_sum(others * scale, red, add);
    const float lse = m + logf(z);

    // the teacher's shares and the row's loss
    float mass = 0.f;
    if (!rest) {
        for (int k = threadIdx.x; k < top; k += kThreads)
            if (share[k] > -INFINITY || share[k] != share[k]) mass += exp_diff(share[k], tmax);
        mass = block_sum(mass, red, add);
    }
    const float norm = rest ? A.teacher_lse[row] : tmax + logf(mass);
    float loss = 0.f, psum = 0.f;
    for (int k = threadIdx.x; k < top; k += kThreads) {
        float p = 0.f;
        if (place[k] >= 0) {
            const float logp = share[k] - norm;
            p = share[k] == -INFINITY ? 0.f : expf(logp);
            if (p != 0.f) loss += p * (logp - (logq[k] - lse));
        }
        share[k] = p;
        psum += p;
    }
    loss = block_sum(loss, red, add);
    psum = block_sum(psum, red, add);
    float inside = psum, outside = psum;
    if (rest) {
        const float pr = fmaxf(0.f, 1.f - psum), qr = others / z;
        if (pr > 0.f && qr > 0.f) {
            loss += pr * (logf(pr) - logf(qr));
            inside = psum + pr;
            outside = inside - pr / qr;
        }
    }
    if (threadIdx.x == 0) A.loss[row] = some > 0.f ? loss * tau * tau : 0.f;
    if (!A.grad) return;
    T* g = static_cast<T*>(A.grad) + row * A.grad_stride;
    const float w = tau * (A.weight ? A.weight[row] : 1.f);
    for (int j = threadIdx.x; j < vocab; j += kThreads) {
        const float v = to_f32(x[j]) * cold;
        g[j] = from_f32<T>(some > 0.f ? w * outside * expf(v - lse) : 0.f);
    }
    __syncthreads();
    // entries: one of those at a place writes for all of them
    for (int k = threadIdx.x; k < top; k += kThreads) {
        const int j = place[k];
        if (j < 0) continue;
        float p = 0.f;
        bool first = true;
        for (int i = 0; i < top; ++i)
            if (place[i] == j) {
                p += share[i];
                if (i < k) first = false;
            }
        if (first) g[j] = from_f32<T>(w * (inside * expf(logq[k] - lse) - p));
    }
}

}  // namespace

hipError_t distill_launch(const hx_distill_args& A) {
    const size_t lds = sizeof(int) * (3 * A.top + (A.vocab + 31) / 32);
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    return with_type(A.type, [&](auto t) {
        return with_type(A.teacher_type, [&](auto u) {
            auto go = [&](auto kernel) {
                if (lds > 65536) {
                    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                             hipFuncAttributeMaxDynamicSharedMemorySize, 163840 - 256);
                    if (e != hipSuccess) return e;
                }
                kernel<<<static_cast<unsigned>(A.rows), kThreads, lds, st>>>(A);
                return hipGetLastError();
            };
            using T = decltype(t);
            using U = decltype(u);
            return A.index_bits == 64 ? go(k_distill<T, U, int64_t>) : go(k_distill<T, U, int32_t>);
        });
    });
}

}  // namespace hx
