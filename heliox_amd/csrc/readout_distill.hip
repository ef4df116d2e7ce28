// The loss against a teacher's top logits, and its gradient by the student's, one workgroup
// per row.
//
// Two passes over a row: the running maximum and sum of a softmax, then the gradient, which
// reads the row again from the cache.  Every place outside the teacher's entries has one factor;
// the few entries are written over afterwards.
//
// Where the rest is one class, the running maximum m_o and the sum z_o are those of the other
// places alone, and the entries are added from their list.  A student that is sure of its
// entries leaves the others a mass q_r far below what fp32 holds beside the largest logit;
// log q_r = (m_o - m) / t + log z_o - log z and the others' gradient
// w (P e^{(m_o - m) / t} / z - p_r / z_o) e^{(x - m_o) / t} have no such limit (z_o is at least 1).
#include "readout.h"

#include <type_traits>

namespace hx {
namespace {

// 2^x by the instruction: one unit off at most, 0 under 2^-126.
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// The k-th of a row's entries: its place (-1: absent), and the teacher's logit.  Indexes and teachers
// of every type go through one kernel: only the few entries are read so.
__device__ __forceinline__ int place_of(const hx_distill_args& A, long long row, int k) {
    const long long at = row * A.index_stride + k;
    const long long j = A.index_bits == 64 ? static_cast<const int64_t*>(A.index)[at] : static_cast<const int32_t*>(A.index)[at];
    return j >= 0 && j < A.vocab ? static_cast<int>(j) : -1;
}

__device__ __forceinline__ float teacher_of(const hx_distill_args& A, long long row, int k) {
    const long long at = row * A.teacher_stride + k;
    switch (A.teacher_type) {
        case HX_F16: return to_f32(static_cast<const __half*>(A.teacher)[at]);
        case HX_BF16: return to_f32(static_cast<const __hip_bfloat16*>(A.teacher)[at]);
        default: return static_cast<const float*>(A.teacher)[at];
    }
}

// LDS: places and teacher's shares of the row's entries, the student's logits there, and, where
// the rest is one class, one bit for each place of the vocabulary that holds an entry.
// Weights are 2^((x - max) cold), cold = log2 e / temperature: the difference comes first, so
// that an error of the product is one of the small difference and not of the logit.  What the
// few entries take, logarithms that nearly cancel, is 64 bits wide; per = 1 / temperature.
template <class T, int kThreads, bool kRest>
__global__ void __launch_bounds__(kThreads, 8) k_distill(hx_distill_args A, float cold, double per) {
    using Vec = typename PieceOf<T>::Vec;
    constexpr int kP = sizeof(Vec) / sizeof(T);
    extern __shared__ int lds[];
    __shared__ double red[kThreads / 64];
    __shared__ float made[3];
    __shared__ int any, twice;               // whether there is an entry, and whether two stand at one place
    const int top = static_cast<int>(A.top), vocab = static_cast<int>(A.vocab);
    int* place = lds;
    float* share = reinterpret_cast<float*>(lds + top);
    float* logit = share + top;
    unsigned* member = reinterpret_cast<unsigned*>(logit + top);
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(A.logits) + row * A.logits_stride;
    const float tau = static_cast<float>(A.temperature);
    auto add = [](auto a, auto b) { return a + b; };
    auto most = [](float a, float b) { return fmaxf(a, b); };
    const float per_f = static_cast<float>(per);
    // fp32 logits have the time for the exact exponential (14 instructions; 16 bits a place have not)
    auto weight = [&](float d) { return sizeof(T) == 4 ? expf(d * per_f) : pow2(d * cold); };

    if constexpr (kRest) {
        for (int w = threadIdx.x; w < (vocab + 31) / 32; w += kThreads) member[w] = 0;
    }
    if (threadIdx.x == 0) any = twice = 0;
    __syncthreads();
    float tmax = -INFINITY, lead = -INFINITY;    // the entries' largest logits, the teacher's and the student's
    for (int k = threadIdx.x; k < top; k += kThreads) {
        const int j = place_of(A, row, k);
        place[k] = j;
        share[k] = j >= 0 ? teacher_of(A, row, k) : -INFINITY;
        logit[k] = j >= 0 ? to_f32(x[j]) : 0.f;
        if (j >= 0) {
            any = 1;
            tmax = fmaxf(tmax, share[k]);
            lead = fmaxf(lead, logit[k]);
            if constexpr (kRest)
                if (atomicOr(member + j / 32, 1u << (j % 32)) >> (j % 32) & 1) twice = 1;
        }
    }
    if constexpr (kRest) lead = block_reduce<kThreads>(lead, red, most);
    else tmax = block_reduce<kThreads>(tmax, red, most);
    const bool some = any;
    double own = 0.;                             // the entries' weights, relative to the largest of them
    if constexpr (kRest) {
        if (lead == -INFINITY) lead = 0.f;
        float mine = 0.f;
        for (int k = threadIdx.x; k < top; k += kThreads) {
            bool counts = place[k] >= 0;
            if (twice)                           // a place counts once
                for (int i = 0; i < k; ++i) counts = counts && place[i] != place[k];
            if (counts) mine += weight(logit[k] - lead);
        }
        own = block_reduce<kThreads>(static_cast<double>(mine), red, add);
    }

    // the student's running maximum and sum over all places, or over those without an entry (bits
    // of `in`: an entry)
    float m = -INFINITY, z = 0.f;
    const int pieces = vocab / kP;
    auto take = [&](float* v, int n, unsigned in) {
        if (kRest && in) {
#pragma unroll
            for (int i = 0; i < kP; ++i)
                if (in >> i & 1) v[i] = -INFINITY;
        }
        float c = v[0];
#pragma unroll
        for (int i = 1; i < kP; ++i)
            if (i < n) c = fmaxf(c, v[i]);
        if (c > m) {
            z *= weight(m - c);                          // m = -inf: 0
            m = c;
        }
        const float from = m == -INFINITY ? 0.f : m;     // nothing but -inf yet: its weights are 0, not NaN
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kP; ++i) sum += i < n ? weight(v[i] - from) : 0.f;
        z += sum;
    };
    const unsigned char* bits = reinterpret_cast<const unsigned char*>(member);
    // f(piece, its logits) for the row's whole pieces, several loads at a time (one alone leaves a
    // CU with 32 KB on their way, less than it takes to keep the memory busy)
    auto each_piece = [&](auto f) {
        constexpr int kAhead = 4;
        for (int p0 = threadIdx.x; p0 < pieces; p0 += kAhead * kThreads) {
            Vec raw[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (p0 + k * kThreads < pieces)
                    raw[k] = *reinterpret_cast<const Vec*>(x + static_cast<long long>(p0 + k * kThreads) * kP);
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (p0 + k * kThreads < pieces) f(p0 + k * kThreads, raw[k]);
        }
    };
    each_piece([&](int p, Vec raw) {
        float v[kP];
#pragma unroll
        for (int i = 0; i < kP; ++i) v[i] = static_cast<float>(raw[i]);
        unsigned in = 0;
        if constexpr (kRest) in = kP == 8 ? bits[p] : bits[p / 2] >> (p % 2 * 4) & 15;
        take(v, kP, in);
    });
    if (pieces * kP + static_cast<int>(threadIdx.x) < vocab) {       // fewer than a piece are left
        const int j = pieces * kP + threadIdx.x;
        float v[kP] = {to_f32(x[j])};
        unsigned in = 0;
        if constexpr (kRest) in = bits[j / 8] >> (j % 8) & 1;
        take(v, 1, in);
    }
    const float mine = m;
    m = block_reduce<kThreads>(m, red, most);
    if (m == -INFINITY) m = 0.f;
    double whole = block_reduce<kThreads>(static_cast<double>(z * weight(mine - m)), red, add);
    const float base = m;                       // what the other places' weights are relative to
    const double beside = whole;                // their sum (0: nothing but -inf)
    // From here to the gradient it is the row as a whole and its entries: waves without entries leave
    // the 64-bit exponentials and logarithms to the others (made by all 16 waves of a row they took
    // 3 to 8% of the call).
    const bool works = threadIdx.x < 64 || static_cast<int>(threadIdx.x) / 64 * 64 < top;
    double under = 1., logz = 0.;               // under: e^{(base - m) / t}
    // (a side that has no weight at all does not count)
    if constexpr (kRest) m = beside == 0. ? lead : own == 0. ? base : fmaxf(base, lead);
    if (works) {
        if constexpr (kRest) {
            const double less = exp((static_cast<double>(fminf(base, lead)) - m) * per);
            under = beside == 0. ? 0. : base < m ? less : 1.;
            whole = beside * under + own * (lead < m ? less : 1.);
        }
        logz = log(whole);
    }

    // the teacher's shares and the row's loss
    double norm;
    if constexpr (kRest) {
        norm = A.teacher_lse[row];
    } else {
        float mass = 0.f;
        for (int k = threadIdx.x; k < top; k += kThreads)
            if (share[k] != -INFINITY) mass += share[k] == tmax ? 1.f : expf((share[k] - tmax) / tau);
        norm = block_reduce<kThreads>(static_cast<double>(mass), red, add);
        if (works) norm = tmax * per + log(norm);
    }
    double loss = 0., psum = 0.;
    for (int k = threadIdx.x; k < top; k += kThreads) {
        float p = 0.f;
        if (share[k] != -INFINITY) {
            const double logp = share[k] * per - norm;
            // 1 - sum p is a share of its own: in 64 bits
            const double wide = kRest ? exp(logp) : static_cast<double>(expf(static_cast<float>(logp)));
            p = static_cast<float>(wide);
            psum += wide;
            if (p != 0.f) loss += p * (logp - ((static_cast<double>(logit[k]) - m) * per - logz));
        }
        share[k] = p;
    }
    loss = block_reduce<kThreads>(loss, red, add);
    psum = block_reduce<kThreads>(psum, red, add);
    if (threadIdx.x < 64) {
        double inside = psum, pull = 0.;        // pull: p_r / z_o
        if constexpr (kRest) {
            const double pr = fmax(0., 1. - psum);
            if (pr > 0. && beside * under > 0.) {   // a mass of 0 in 64 bits is that of masked places
                loss += pr * (log(pr / beside) - ((static_cast<double>(base) - m) * per - logz));
                inside = psum + pr;
                pull = pr / beside;
            }
        }
        if (threadIdx.x == 0) {
            A.loss[row] = some ? static_cast<float>(loss * tau * tau) : 0.f;
            made[0] = some ? tau * (A.weight ? A.weight[row] : 1.f) : 0.f;
            made[1] = static_cast<float>(made[0] * (inside * under / whole - pull));
            made[2] = static_cast<float>(inside / whole);
        }
    }
    if (!A.grad) return;
    __syncthreads();
    T* g = static_cast<T*>(A.grad) + row * A.grad_stride;
    const float w = made[0], factor = made[1], within = made[2];
    // (entries may lie far above the base; theirs are written over below)
    auto slope = [&](float v) { return some ? factor * weight(v - base) : 0.f; };
    each_piece([&](int p, Vec raw) {
#pragma unroll
        for (int i = 0; i < kP; ++i) raw[i] = static_cast<decltype(raw[0] + raw[0])>(slope(static_cast<float>(raw[i])));
        *reinterpret_cast<Vec*>(g + static_cast<long long>(p) * kP) = raw;
    });
    if (pieces * kP + static_cast<int>(threadIdx.x) < vocab) {
        const int j = pieces * kP + threadIdx.x;
        g[j] = from_f32<T>(slope(to_f32(x[j])));
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
        if (first) g[j] = from_f32<T>(w * (within * weight(logit[k] - m) - p));
    }
}

template <class T, int kThreads, bool kRest>
hipError_t launch(const hx_distill_args& A) {
    const size_t lds = sizeof(int) * (3 * A.top + (kRest ? (A.vocab + 31) / 32 : 0));
    auto kernel = k_distill<T, kThreads, kRest>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, 163840 - 256);
        if (e != hipSuccess) return e;
    }
    kernel<<<static_cast<unsigned>(A.rows), kThreads, lds, static_cast<hipStream_t>(A.stream)>>>(
        A, static_cast<float>(1.4426950408889634 / A.temperature), 1.0 / A.temperature);
    return hipGetLastError();
}

template <class T>
hipError_t pick(const hx_distill_args& A) {
    // Threads a row.  A CU holds 2048: rows of a last, thin round run alone, so 512 threads
    // where that fits all rows into one round and 1024 does not (517 rows of 50021: 48 us with
    // 1024, 38 with 512); small rows take no more than they have pieces for.
    const bool small = A.vocab <= 4096, half = A.rows > 512 && A.rows <= 1024;
    auto go = [&](auto rest) {
        constexpr bool kRest = decltype(rest)::value;
        return small  ? launch<T, 256, kRest>(A)
               : half ? launch<T, 512, kRest>(A)
                      : launch<T, 1024, kRest>(A);
    };
    return A.teacher_lse ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

hipError_t distill_launch(const hx_distill_args& A) {
    return with_type(A.type, [&](auto t) { return pick<decltype(t)>(A); });
}

}  // namespace hx
