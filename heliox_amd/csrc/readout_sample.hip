// The drawing of an answer from logits, one workgroup per row.  Masses are whole numbers, so
// their sums are the same in any order.
#include "readout.h"

namespace hx {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr float kMass = 1099511627776.f;      // 2^40
typedef unsigned long long u64;

// Order-preserving key of a logit: larger key, larger logit; -0 and 0 alike, NaN as -inf.
__device__ __forceinline__ unsigned key_of(float x) {
    if (x != x) x = -INFINITY;
    const unsigned u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Shared {
    u64 bins[256];
    u64 part[kWaves];
    u64 pick[3];
};

__device__ u64 block_sum(u64 x, Shared& sh) {
    for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
    __syncthreads();
    if (threadIdx.x % 64 == 0) sh.part[threadIdx.x / 64] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kWaves; ++w) x += sh.part[w];
    return x;
}

// Sum of x over the threads before this one; total gets the whole sum.
__device__ u64 block_before(u64 x, Shared& sh, u64& total) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    u64 run = x;
    for (int m = 1; m < 64; m <<= 1) {
        const u64 other = __shfl_up(run, m);
        if (lane >= m) run += other;
    }
    __syncthreads();
    if (lane == 63) sh.part[wave] = run;
    __syncthreads();
    u64 before = 0;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += sh.part[w];
        total += sh.part[w];
    }
    return before + run - x;
}

template <class T>
struct Row {
    const T* x;
    int n;
    unsigned top;       // key of the largest
    float most, cold;   // the largest logit, 1 / temperature

    __device__ unsigned key(int j) const { return key_of(to_f32(x[j])); }
    __device__ float weight(unsigned k) const {
        return k == top ? 1.f : expf((value_of(k) - most) * cold);
    }
    __device__ u64 mass(unsigned k) const { return static_cast<u64>(weight(k) * kMass); }
};

// The key at which a running sum over the places in descending order passes a bound: value(key)
// is what a place counts, passes(sum) whether a sum reaches the bound.  before gets the sum
// over larger keys.  Places with a key under `least` are left out.
template <class T, class V, class P>
__device__ unsigned select(const Row<T>& R, unsigned least, Shared& sh, V value, P passes, u64& before) {
    unsigned prefix = 0, mask = 0;
    before = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) sh.bins[threadIdx.x] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < R.n; j += kThreads) {
            const unsigned k = R.key(j);
            if (k >= least && (k & mask) == prefix) atomicAdd(&sh.bins[k >> shift & 255], value(k));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 sum = before;
            int bin = 255;
            while (bin > 0 && !passes(sum + sh.bins[bin])) sum += sh.bins[bin--];
            sh.pick[0] = bin;
            sh.pick[1] = sum;
        }
        __syncthreads();
        prefix |= static_cast<unsigned>(sh.pick[0]) << shift;
        mask |= 255u << shift;
        before = sh.pick[1];
    }
    return prefix;
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sample(hx_sample_args A) {
    __shared__ Shared sh;
    const long long row = blockIdx.x;
    Row<T> R;
    R.x = static_cast<const T*>(A.logits) + row * A.logits_stride;
    R.n = static_cast<int>(A.vocab);
    const float temp = A.temperature ? A.temperature[row] : static_cast<float>(A.temperature_value);
    long long top_k = A.top_k ? A.top_k[row] : A.top_k_value;
    const float top_p = A.top_p ? A.top_p[row] : static_cast<float>(A.top_p_value);
    const float min_p = fminf(A.min_p ? A.min_p[row] : static_cast<float>(A.min_p_value), 1.f);
    const bool greedy = !(temp > 0.f);
    if (greedy) top_k = 1;
    R.cold = greedy ? 1.f : 1.f / temp;
    unsigned best = 0;
    for (int j = threadIdx.x; j < R.n; j += kThreads) best = max(best, R.key(j));
    for (int m = 32; m > 0; m >>= 1) best = max(best, __shfl_xor(best, m));
    if (threadIdx.x % 64 == 0) sh.part[threadIdx.x / 64] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = max(best, static_cast<unsigned>(sh.part[w]));
    R.top = best;
    R.most = value_of(best);
    if (R.most == -INFINITY) {
        if (threadIdx.x == 0) {
            A.token[row] = -1;
            A.logprob[row] = -INFINITY;
        }
        return;
    }
    // Places stay whose key is over `least`, and the first `ties` by index of those at it.
    unsigned least = 0;
    u64 ties = R.n;
    if (top_k > 0 && top_k < R.n) {
        u64 before;
        least = select(R, 0u, sh, [](unsigned) { return u64(1); },
                       [&](u64 n) { return n >= static_cast<u64>(top_k); }, before);
        ties = top_k - before;
    }
    auto counted = [&](unsigned k) { return k >= least ? R.mass(k) : 0; };
    if (!(top_p >= 1.f)) {
        u64 above = 0, at = 0;
        for (int j = threadIdx.x; j < R.n; j += kThreads) {
            const unsigned k = R.key(j);
            if (k > least) above += R.mass(k);
            if (k == least) ++at;
        }
        above = block_sum(above, sh);
        at = min(block_sum(at, sh), ties);
        const double sum = static_cast<double>(above + at * (at ? R.mass(least) : 0));
        const double bound = fmax(static_cast<double>(top_p) * sum, 0.5);    // the largest stays
        // the last place that stays is the last with less than the bound before it
        u64 before;
        const unsigned cut = select(R, least, sh, counted,
                                    [&](u64 s) { return static_cast<double>(s) >= bound; }, before);
        if (cut > least) ties = R.n;
        least = cut;
        const u64 m = R.mass(least);
        u64 lo = 1, hi = max(ties, u64(1));    // the first at the cut stays: its sum before is under the bound
        while (lo < hi) {
            const u64 mid = (lo + hi + 1) / 2;
            if (static_cast<double>(before + (mid - 1) * m) < bound) lo = mid;
            else hi = mid - 1;
        }
        ties = lo;
    }
    // The kept mass, then the place where its running sum passes u of it, in index order.
    auto kept = [&](int j, u64& tie) {
        const unsigned k = j < R.n ? R.key(j) : 0;
        tie = j < R.n && k == least;
        return j < R.n && k >= least && R.weight(k) >= min_p ? R.mass(k) : 0;
    };
    u64 total = 0, seen = 0;
    for (int pass = 0; pass < 2; ++pass) {
        const double u = fmin(fmax(static_cast<double>(A.u[row]), 0.0), 1.0);
        const u64 aim = pass ? min(static_cast<u64>(floor(u * static_cast<double>(total))), total - 1) : 0;
        u64 sum = 0;
        seen = 0;
        for (int j0 = 0; j0 < R.n; j0 += kThreads) {
            const int j = j0 + threadIdx.x;
            u64 tie, tied, whole;
            u64 m = kept(j, tie);
            const u64 rank = seen + block_before(tie, sh, tied);
            if (tie && rank >= ties) m = 0;
            const u64 before = sum + block_before(m, sh, whole);
            if (pass && m && before <= aim && aim < before + m) {
                A.token[row] = j;
                const unsigned k = R.key(j);
                const float z = k == R.top ? 0.f : (value_of(k) - R.most) * R.cold;
                A.logprob[row] = z - logf(static_cast<float>(total) / kMass);
            }
            seen += tied;
            sum += whole;
        }
        if (!pass) total = sum;
    }
}

}  // namespace

hipError_t sample_launch(const hx_sample_args& A) {
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    return with_type(A.type, [&](auto t) {
        k_sample<decltype(t)><<<static_cast<unsigned>(A.rows), kThreads, 0, st>>>(A);
        return hipGetLastError();
    });
}

}  // namespace hx
