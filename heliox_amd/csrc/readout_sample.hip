// The drawing of an answer from logits, one workgroup per row.
//
// Masses are whole numbers, so their sums are the same in any order, and integer atomics may
// make them.  What top_k and top_p leave is "every place over a key, and the first of those at
// it by index"; the key is found from histograms: one over places in 2048 equal parts of the
// range that has any mass, then over the keys of the one part where the sum passes the bound.
// Where top_k leaves at most as many places as the workgroup has threads, those go into LDS and
// are sorted there instead.  The row itself is read again from the cache in each pass.
#include "readout.h"

namespace hx {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr float kMass = 1099511627776.f;      // 2^40
constexpr float kDepth = 27.8f;               // e^-27.8 < 2^-40: no mass beyond
typedef unsigned long long u64;

template <class T> struct PieceOf;
template <> struct PieceOf<float> { typedef float Vec __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct PieceOf<__half> { typedef _Float16 Vec __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct PieceOf<__hip_bfloat16> { typedef __bf16 Vec __attribute__((ext_vector_type(8), aligned(2))); };

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
    u64 bins[kBins];
    u64 part[kWaves];
    u64 pick[2];
    unsigned count;
};

// x reduced over the workgroup; every thread gets the result.
template <class V, class F>
__device__ __forceinline__ V block_reduce(V x, Shared& sh, F op) {
    for (int m = 32; m > 0; m >>= 1) x = op(x, __shfl_xor(x, m));
    __syncthreads();
    if (threadIdx.x % 64 == 0) sh.part[threadIdx.x / 64] = x;
    __syncthreads();
    x = static_cast<V>(sh.part[0]);
    for (int w = 1; w < kWaves; ++w) x = op(x, static_cast<V>(sh.part[w]));
    return x;
}

__device__ __forceinline__ u64 block_sum(u64 x, Shared& sh) {
    return block_reduce(x, sh, [](u64 a, u64 b) { return a + b; });
}

__device__ __forceinline__ u64 wave_before(u64 x) {       // sum over the lanes before this one
    const int lane = threadIdx.x % 64;
    u64 run = x;
    for (int m = 1; m < 64; m <<= 1) {
        const u64 other = __shfl_up(run, m);
        if (lane >= m) run += other;
    }
    return run - x;
}

// Sum of x over the threads before this one; total gets the whole sum.
__device__ u64 block_before(u64 x, Shared& sh, u64& total) {
    const u64 before = wave_before(x);
    __syncthreads();
    if (threadIdx.x % 64 == 63) sh.part[threadIdx.x / 64] = before + x;
    __syncthreads();
    u64 base = 0;
    total = 0;
    for (int w = 0; w < kWaves; ++w) {
        if (w < static_cast<int>(threadIdx.x / 64)) base += sh.part[w];
        total += sh.part[w];
    }
    return base + before;
}

template <class T>
struct Row {
    using Vec = typename PieceOf<T>::Vec;
    static constexpr int kP = sizeof(Vec) / sizeof(T);
    const T* x;
    int n;
    float most, cold;   // the largest logit, 1 / temperature

    // f(first index, kP logits, how many of them are there) for the pieces of the row; piece p is
    // thread p % kThreads's.  All threads of a wave take as many turns.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        const int whole = n / kP, pieces = (n + kP - 1) / kP;
        for (int p0 = 0; p0 < pieces; p0 += kThreads) {
            const int p = p0 + threadIdx.x;
            float v[kP];
            if (p < whole) {
                const Vec raw = *reinterpret_cast<const Vec*>(x + static_cast<long long>(p) * kP);
#pragma unroll
                for (int i = 0; i < kP; ++i) v[i] = static_cast<float>(raw[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kP; ++i) v[i] = p * kP + i < n ? to_f32(x[p * kP + i]) : -INFINITY;
            }
            f(p * kP, v, max(0, min(kP, n - p * kP)));
        }
    }
    __device__ __forceinline__ float depth(float v) const {     // of a logit under the largest, over the temperature
        return v == most ? 0.f : (v - most) * cold;
    }
    __device__ __forceinline__ float weight(float v) const { return expf(depth(v)); }
    __device__ __forceinline__ u64 mass(float v) const { return static_cast<u64>(weight(v) * kMass); }
};

// Of sh.bins from the last to the first, the one where the running sum (from `before`) passes;
// before gets the sum up to it, and the whole sum is returned where none passes (bin -1).
template <class P>
__device__ int find_bin(Shared& sh, P passes, u64& before) {
    __syncthreads();
    constexpr int kEach = kBins / kThreads;
    const int top = kBins - 1 - threadIdx.x * kEach;
    u64 mine = 0, total;
    for (int i = 0; i < kEach; ++i) mine += sh.bins[top - i];
    u64 sum = before + block_before(mine, sh, total);
    if (threadIdx.x == 0) {
        sh.pick[0] = ~0ull;
        sh.pick[1] = before + total;
    }
    __syncthreads();
    if (!passes(sum) && passes(sum + mine))
        for (int i = 0; i < kEach; ++i) {
            if (passes(sum + sh.bins[top - i])) {
                sh.pick[0] = top - i;
                sh.pick[1] = sum;
                break;
            }
            sum += sh.bins[top - i];
        }
    __syncthreads();
    const int bin = static_cast<int>(static_cast<long long>(sh.pick[0]));
    before = sh.pick[1];
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    return bin;
}

// The key at which a running sum over the places in descending order passes a bound: value(v)
// is what a place counts (0: nothing), passes(sum) whether a sum reaches the bound.  before gets
// the sum over larger keys.  Returns 0 where all places with a mass do not reach the bound.
// sh.bins are zero before and after.
template <class T, class V, class P>
__device__ unsigned select(const Row<T>& R, Shared& sh, V value, P passes, u64& before) {
    // equal parts of the depth; monotonous, as each rounding is
    auto part = [&](float v) {
        const float d = -R.depth(v) * (kBins / kDepth);
        return d < kBins ? kBins - 1 - static_cast<int>(d) : -1;
    };
    R.each([&](int, const float* v, int n) {
#pragma unroll
        for (int i = 0; i < Row<T>::kP; ++i) {
            const int b = i < n ? part(v[i]) : -1;
            if (b >= 0) {
                const u64 w = value(v[i]);
                if (w) atomicAdd(&sh.bins[b], w);
            }
        }
    });
    before = 0;
    const int bin = find_bin(sh, passes, before);
    if (bin < 0) return 0;
    // the part's keys: least and largest, then 2048 parts of what lies between, until one key is left
    unsigned lo = ~0u, hi = 0;
    R.each([&](int, const float* v, int n) {
#pragma unroll
        for (int i = 0; i < Row<T>::kP; ++i)
            if (i < n && part(v[i]) == bin && value(v[i])) {
                const unsigned k = key_of(v[i]);
                lo = min(lo, k);
                hi = max(hi, k);
            }
    });
    lo = block_reduce(lo, sh, [](unsigned a, unsigned b) { return min(a, b); });
    hi = block_reduce(hi, sh, [](unsigned a, unsigned b) { return max(a, b); });
    while (lo < hi) {
        int shift = 0;
        while ((hi - lo) >> shift >= kBins) ++shift;
        __syncthreads();
        R.each([&](int, const float* v, int n) {
#pragma unroll
            for (int i = 0; i < Row<T>::kP; ++i)
                if (i < n) {
                    const unsigned k = key_of(v[i]);
                    if (k >= lo && k <= hi) {
                        const u64 w = value(v[i]);
                        if (w) atomicAdd(&sh.bins[(k - lo) >> shift], w);
                    }
                }
        });
        const int b = find_bin(sh, passes, before);
        lo += static_cast<unsigned>(b) << shift;
        hi = min(hi, lo + ((1u << shift) - 1));
    }
    return lo;
}

// Ascending sort of kThreads keys, one a thread, in LDS.
__device__ u64 block_sort(u64 key, u64* at) {
    for (int size = 2; size <= kThreads; size <<= 1)
        for (int gap = size / 2; gap > 0; gap >>= 1) {
            u64 other;
            if (gap >= 64) {
                __syncthreads();
                at[threadIdx.x] = key;
                __syncthreads();
                other = at[threadIdx.x ^ gap];
            } else {
                other = __shfl_xor(key, gap);
            }
            const bool low = (threadIdx.x & gap) == 0, up = (threadIdx.x & size) == 0;
            key = (key < other) == (low == up) ? key : other;
        }
    return key;
}

// How many places at a key stay: those with less than the bound before them, of at most n.
__device__ u64 count_under(double bound, u64 before, u64 mass, u64 n) {
    u64 lo = 1, hi = n > 1 ? n : 1;
    while (lo < hi) {
        const u64 mid = (lo + hi + 1) / 2;
        if (static_cast<double>(before + (mid - 1) * mass) < bound) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ u64 aim_of(float u, u64 total) {
    const double share = fmin(fmax(static_cast<double>(u), 0.0), 1.0);
    const u64 aim = static_cast<u64>(floor(share * static_cast<double>(total)));
    return aim < total ? aim : total - 1;
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sample(hx_sample_args A) {
    __shared__ Shared sh;
    extern __shared__ u64 segments[];          // mass of each wave's turn in each()
    using R_ = Row<T>;
    constexpr int kP = R_::kP;
    const long long row = blockIdx.x;
    R_ R;
    R.x = static_cast<const T*>(A.logits) + row * A.logits_stride;
    R.n = static_cast<int>(A.vocab);
    const float temp = A.temperature ? A.temperature[row] : static_cast<float>(A.temperature_value);
    long long top_k = A.top_k ? A.top_k[row] : A.top_k_value;
    const float top_p = A.top_p ? A.top_p[row] : static_cast<float>(A.top_p_value);
    const float min_p = fminf(A.min_p ? A.min_p[row] : static_cast<float>(A.min_p_value), 1.f);
    const bool greedy = !(temp > 0.f);
    if (greedy) top_k = 1;
    if (top_k >= R.n) top_k = 0;
    R.cold = greedy ? 1.f : 1.f / temp;
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    if (threadIdx.x == 0) sh.count = 0;

    float most = -INFINITY;                    // fmaxf passes over NaN
    R.each([&](int, const float* v, int) {
#pragma unroll
        for (int i = 0; i < kP; ++i) most = fmaxf(most, v[i]);
    });
    R.most = value_of(block_reduce(key_of(most), sh, [](unsigned a, unsigned b) { return max(a, b); }));
    auto answer = [&](int j, float v, u64 total) {
        A.token[row] = j;
        A.logprob[row] = R.depth(v) - logf(static_cast<float>(total) / kMass);
    };
    if (R.most == -INFINITY) {
        if (threadIdx.x == 0) {
            A.token[row] = -1;
            A.logprob[row] = -INFINITY;
        }
        return;
    }

    // Places stay whose key is over `least`, and the first `ties` by index of the `at` at it.
    unsigned least = 0;
    u64 ties = R.n, at = R.n;
    if (top_k > 0) {
        u64 before;
        least = select(R, sh, [](float v) { return u64(v == v); },
                       [&](u64 n) { return n >= static_cast<u64>(top_k); }, before);
        if (least) ties = top_k - before;
        // (where fewer than top_k places have a mass, all that have one stay)
    }
    if (top_k > 0 && top_k <= kThreads) {
        // those places into LDS, in whatever order
        u64* const list = sh.bins;
        static_assert(kBins >= 2 * kThreads, "the list and the sort's own space");
        R.each([&](int j0, const float* v, int n) {
#pragma unroll
            for (int i = 0; i < kP; ++i)
                if (i < n && R.mass(v[i])) {
                    const unsigned k = key_of(v[i]);
                    if (k > least) list[atomicAdd(&sh.count, 1u)] = static_cast<u64>(~k) << 32 | (j0 + i);
                }
        });
        __syncthreads();
        const unsigned first = sh.count;
        // the first `ties` by index of those at the key: by their rank among the row's
        u64 seen = 0;
        if (least)
            R.each([&](int j0, const float* v, int n) {
                unsigned mine = 0;
#pragma unroll
                for (int i = 0; i < kP; ++i) mine += i < n && v[i] == v[i] && key_of(v[i]) == least;
                if (seen >= ties) return;      // the same for all threads
                u64 turn;
                u64 rank = seen + block_before(mine, sh, turn);
                seen += turn;
#pragma unroll
                for (int i = 0; i < kP; ++i)
                    if (i < n && v[i] == v[i] && key_of(v[i]) == least) {
                        if (rank < ties) list[first + rank] = static_cast<u64>(~least) << 32 | (j0 + i);
                        ++rank;
                    }
            });
        __syncthreads();
        const unsigned count = first + static_cast<unsigned>(least ? ties : 0);
        u64 key = threadIdx.x < count ? list[threadIdx.x] : ~0ull;
        __syncthreads();
        key = block_sort(key, list + kThreads);
        // in rank order now
        const bool there = threadIdx.x < count;
        const float v = there ? value_of(~static_cast<unsigned>(key >> 32)) : -INFINITY;
        u64 m = there ? R.mass(v) : 0, total;
        u64 before = block_before(m, sh, total);
        if (!(top_p >= 1.f)) {
            const double bound = fmax(static_cast<double>(top_p) * static_cast<double>(total), 0.5);
            if (!(static_cast<double>(before) < bound)) m = 0;
        }
        if (there && !(R.weight(v) >= min_p)) m = 0;
        // and in index order
        key = block_sort(m ? key << 32 | key >> 32 : ~0ull, list + kThreads);
        const bool stays = key != ~0ull;
        const float w = stays ? value_of(~static_cast<unsigned>(key)) : -INFINITY;
        m = stays ? R.mass(w) : 0;
        before = block_before(m, sh, total);
        const u64 aim = aim_of(A.u[row], total);
        if (m && before <= aim && aim < before + m) answer(static_cast<int>(key >> 32), w, total);
        return;
    }

    if (!(top_p >= 1.f)) {
        auto counted = [&](float v) { return key_of(v) >= least ? R.mass(v) : 0; };
        u64 over = 0, same = 0;
        R.each([&](int, const float* v, int n) {
#pragma unroll
            for (int i = 0; i < kP; ++i)
                if (i < n) {
                    const unsigned k = key_of(v[i]);
                    if (k > least) over += R.mass(v[i]);
                    same += k == least;
                }
        });
        over = block_sum(over, sh);
        at = block_sum(same, sh);
        const u64 stay = min(at, ties);
        const u64 m_least = least ? R.mass(value_of(least)) : 0;
        // the largest stays whatever the bound is
        const double bound = fmax(static_cast<double>(top_p) * static_cast<double>(over + stay * m_least), 0.5);
        u64 before;
        const unsigned cut = select(R, sh, counted, [&](u64 s) { return static_cast<double>(s) >= bound; }, before);
        ties = count_under(bound, before, R.mass(value_of(cut)), cut > least ? R.n : stay);
        least = cut;
    }
    // Only some of the places at the key stay: up to which index?
    int last = R.n;
    if (least) {
        u64 seen = 0;
        int found = R.n;
        R.each([&](int j0, const float* v, int n) {
            if (seen >= ties) return;          // the same for all threads
            unsigned mine = 0;
#pragma unroll
            for (int i = 0; i < kP; ++i) mine += i < n && key_of(v[i]) == least;
            u64 turn;
            u64 rank = seen + block_before(mine, sh, turn);
            seen += turn;
#pragma unroll
            for (int i = 0; i < kP; ++i)
                if (i < n && key_of(v[i]) == least && ++rank == ties) found = j0 + i;
        });
        last = block_reduce(found, sh, [](int a, int b) { return min(a, b); });
    }
    auto kept = [&](int j, float v) -> u64 {
        const unsigned k = key_of(v);
        const float w = R.weight(v);
        return (k > least || (k == least && j <= last)) && w >= min_p ? static_cast<u64>(w * kMass) : 0;
    };
    // What stays of each wave's turns, their running sum, and in the turn where it passes u of
    // the whole the place itself.
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    int turn = 0;
    R.each([&](int j0, const float* v, int n) {
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < kP; ++i) m += i < n ? kept(j0 + i, v[i]) : 0;
        for (int s = 32; s > 0; s >>= 1) m += __shfl_xor(m, s);
        if (lane == 0) segments[turn * kWaves + wave] = m;
        ++turn;
    });
    __syncthreads();
    const int nseg = turn * kWaves, per = (nseg + kThreads - 1) / kThreads;
    const int s0 = min(static_cast<int>(threadIdx.x) * per, nseg), s1 = min(s0 + per, nseg);
    u64 mine = 0, total;
    for (int s = s0; s < s1; ++s) mine += segments[s];
    u64 before = block_before(mine, sh, total);
    const u64 aim = aim_of(A.u[row], total);
    if (mine && before <= aim && aim < before + mine) {
        int s = s0;
        while (before + segments[s] <= aim) before += segments[s++];
        sh.pick[0] = s;
        sh.pick[1] = before;
    }
    __syncthreads();
    if (wave != 0) return;
    const int seg = static_cast<int>(sh.pick[0]);
    const int j0 = ((seg / kWaves) * kThreads + seg % kWaves * 64 + lane) * kP;
    u64 m[kP], sum = 0;
    float v[kP];
#pragma unroll
    for (int i = 0; i < kP; ++i) {
        v[i] = j0 + i < R.n ? to_f32(R.x[j0 + i]) : -INFINITY;
        m[i] = j0 + i < R.n ? kept(j0 + i, v[i]) : 0;
        sum += m[i];
    }
    before = sh.pick[1] + wave_before(sum);
#pragma unroll
    for (int i = 0; i < kP; ++i) {
        if (m[i] && before <= aim && aim < before + m[i]) answer(j0 + i, v[i], total);
        before += m[i];
    }
}

}  // namespace

hipError_t sample_launch(const hx_sample_args& A) {
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        constexpr int64_t turn = static_cast<int64_t>(kThreads) * Row<T>::kP;
        const size_t lds = sizeof(u64) * kWaves * ((A.vocab + turn - 1) / turn);
        if (lds > 32768) {
            const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_sample<T>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, 140000);
            if (e != hipSuccess) return e;
        }
        k_sample<T><<<static_cast<unsigned>(A.rows), kThreads, lds, st>>>(A);
        return hipGetLastError();
    });
}

}  // namespace hx
