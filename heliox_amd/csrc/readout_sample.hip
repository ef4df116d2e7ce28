// The drawing of an answer from logits, one workgroup per row.
//
// Masses are whole numbers, so their sums are the same in any order, and integer atomics may
// make them.  What top_k and top_p leave is "every place over a key, and those at it up to an
// index".  A histogram over equal parts (two a thread) of the range that has any mass says in
// which part the cut lies; the places of that part (and, for top_k, of all above) go into LDS
// where they fit, are sorted there and say the rest.  Where they do not fit (ties without end), histograms
// over the part's keys go on until one key is left.  The row itself is read again from the cache
// in each pass: two to four of them as a rule, of which those that make masses of all places
// (about 40 instructions each) take the time: 256 rows of 131072 bf16 logits, each with its own
// settings, take 121 us, nine times what reading them once would, 16 waves a CU busy throughout.
#include "readout.h"

#include <type_traits>

namespace hx {
namespace {

constexpr float kMass = 1099511627776.f;      // 2^40
constexpr float kDepth = 27.8f;               // e^-27.8 < 2^-40: no mass beyond
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

template <int kT>
struct Shared {
    static constexpr int kThreads = kT, kWaves = kT / 64, kBins = 2 * kT;
    u64 bins[kBins];
    u64 part[kWaves];
    u64 pick[3];
    unsigned count;
};

template <class Sh>
__device__ __forceinline__ u64 block_sum(u64 x, Sh& sh) {
    return block_reduce<Sh::kThreads>(x, sh.part, [](u64 a, u64 b) { return a + b; });
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
template <class Sh>
__device__ __forceinline__ u64 block_before(u64 x, Sh& sh, u64& total) {
    const u64 before = wave_before(x);
    __syncthreads();
    if (threadIdx.x % 64 == 63) sh.part[threadIdx.x / 64] = before + x;
    __syncthreads();
    u64 base = 0;
    total = 0;
    for (int w = 0; w < Sh::kWaves; ++w) {
        if (w < static_cast<int>(threadIdx.x / 64)) base += sh.part[w];
        total += sh.part[w];
    }
    return base + before;
}

template <class T, int kThreads>
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

struct Cut {
    int bin;            // -1: the bound is not reached
    u64 before, at;     // the sums over what comes before it, and of it
};

// Of sh.bins from the last to the first, the one where the running sum (from `before`) passes.
// The bins are zero afterwards.
template <class Sh, class P>
__device__ __forceinline__ Cut find_bin(Sh& sh, P passes, u64 before) {
    constexpr int kThreads = Sh::kThreads, kBins = Sh::kBins;
    __syncthreads();
    constexpr int kEach = kBins / kThreads;
    const int top = kBins - 1 - threadIdx.x * kEach;
    u64 mine = 0, total;
    for (int i = 0; i < kEach; ++i) mine += sh.bins[top - i];
    u64 sum = before + block_before(mine, sh, total);
    if (threadIdx.x == 0) sh.pick[0] = ~0ull;
    __syncthreads();
    if (!passes(sum) && passes(sum + mine))
        for (int i = 0; i < kEach; ++i) {
            if (passes(sum + sh.bins[top - i])) {
                sh.pick[0] = top - i;
                sh.pick[1] = sum;
                sh.pick[2] = sh.bins[top - i];
                break;
            }
            sum += sh.bins[top - i];
        }
    __syncthreads();
    const Cut c{static_cast<int>(static_cast<long long>(sh.pick[0])), sh.pick[1], sh.pick[2]};
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    return c;
}

// Which of the equal parts of the range with any mass a logit lies in, the largest in the last;
// -1: beyond.  Monotonous, as each of its roundings is.
template <int kBins, class R_>
__device__ __forceinline__ int part_of(const R_& R, float v) {
    const float d = -R.depth(v) * (kBins / kDepth);
    return d < kBins ? kBins - 1 - static_cast<int>(d) : -1;
}

// Adds value(index, logit) to the bin of each place's part.
template <class R_, class Sh, class V>
__device__ __forceinline__ void add_parts(const R_& R, Sh& sh, V value) {
    R.each([&](int j0, const float* v, int n) {
#pragma unroll
        for (int i = 0; i < R_::kP; ++i) {
            const int b = i < n ? part_of<Sh::kBins>(R, v[i]) : -1;
            if (b >= 0) {
                const u64 w = value(j0 + i, v[i]);
                if (w) atomicAdd(&sh.bins[b], w);
            }
        }
    });
}

// From the part where a running sum passes to the key where it does: by histograms over what
// lies between the part's least and largest key, until one key is left.  c is the part's cut
// and becomes the key's.
template <class R_, class Sh, class V, class P>
__device__ __forceinline__ unsigned refine(const R_& R, Sh& sh, V value, P passes, Cut& c) {
    constexpr int kBins = Sh::kBins;
    unsigned lo = ~0u, hi = 0;
    R.each([&](int j0, const float* v, int n) {
#pragma unroll
        for (int i = 0; i < R_::kP; ++i)
            if (i < n && part_of<kBins>(R, v[i]) == c.bin && value(j0 + i, v[i])) {
                const unsigned k = key_of(v[i]);
                lo = min(lo, k);
                hi = max(hi, k);
            }
    });
    lo = block_reduce<Sh::kThreads>(lo, sh.part, [](unsigned a, unsigned b) { return min(a, b); });
    hi = block_reduce<Sh::kThreads>(hi, sh.part, [](unsigned a, unsigned b) { return max(a, b); });
    while (lo < hi) {
        int shift = 0;
        while ((hi - lo) >> shift >= kBins) ++shift;
        R.each([&](int j0, const float* v, int n) {
#pragma unroll
            for (int i = 0; i < R_::kP; ++i) {
                const unsigned k = key_of(v[i]);
                if (i < n && k >= lo && k <= hi) {
                    const u64 w = value(j0 + i, v[i]);
                    if (w) atomicAdd(&sh.bins[(k - lo) >> shift], w);
                }
            }
        });
        c = find_bin(sh, passes, c.before);
        lo += static_cast<unsigned>(c.bin) << shift;
        hi = min(hi, lo + ((1u << shift) - 1));
    }
    return lo;
}

// Ascending sort of kThreads keys, one a thread, in LDS.
template <int kThreads>
__device__ __forceinline__ u64 block_sort(u64 key, u64* at) {
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

constexpr u64 kNone = ~0ull;
__device__ __forceinline__ u64 by_rank(float v, int j) { return static_cast<u64>(~key_of(v)) << 32 | static_cast<unsigned>(j); }
__device__ __forceinline__ float ranked_value(u64 e) { return value_of(~static_cast<unsigned>(e >> 32)); }

// The places for which take(index, logit) holds, sorted by rank, one a thread (kNone: no more);
// false, and nothing usable, where they are more than the threads.  Uses sh.bins.
template <class R_, class Sh, class F>
__device__ __forceinline__ bool gather(const R_& R, Sh& sh, F take, u64& mine) {
    constexpr int kThreads = Sh::kThreads, kBins = Sh::kBins;
    u64* const list = sh.bins;
    static_assert(kBins >= 2 * kThreads, "the list and the sort's own space");
    R.each([&](int j0, const float* v, int n) {
#pragma unroll
        for (int i = 0; i < R_::kP; ++i)
            if (i < n && take(j0 + i, v[i])) {
                const unsigned at = atomicAdd(&sh.count, 1u);
                if (at < kThreads) list[at] = by_rank(v[i], j0 + i);
            }
    });
    __syncthreads();
    const unsigned count = sh.count;
    mine = threadIdx.x < min(count, static_cast<unsigned>(kThreads)) ? list[threadIdx.x] : kNone;
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    if (count <= kThreads) mine = block_sort<kThreads>(mine, list + kThreads);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) list[i] = 0;
    __syncthreads();
    return count <= kThreads;
}

// How many places at a key stay: those with less than the bound before them, of at most n.
__device__ __forceinline__ u64 count_under(double bound, u64 before, u64 mass, u64 n) {
    u64 lo = 1, hi = n > 1 ? n : 1;
    while (lo < hi) {
        const u64 mid = (lo + hi + 1) / 2;
        if (static_cast<double>(before + (mid - 1) * mass) < bound) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The place where the running sum of value(index, logit), in index order, passes an aim: each
// wave's turns are summed, then the turn where it passes is looked at by itself.  aim_of(whole
// sum) is the aim; found(index, logit, whole sum) is called by the one thread that holds the place.
template <class R_, class Sh, class V, class A, class F>
__device__ __forceinline__ void at_running_sum(const R_& R, Sh& sh, u64* segments, V value, A aim_of, F found) {
    constexpr int kP = R_::kP, kThreads = Sh::kThreads, kWaves = Sh::kWaves;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    int turn = 0;
    R.each([&](int j0, const float* v, int n) {
        u64 m = 0;
#pragma unroll
        for (int i = 0; i < kP; ++i) m += i < n ? value(j0 + i, v[i]) : 0;
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
    const u64 aim = aim_of(total);
    if (mine && before <= aim && aim < before + mine) {
        int s = s0;
        while (before + segments[s] <= aim) before += segments[s++];
        sh.pick[0] = s;
        sh.pick[1] = before;
    }
    __syncthreads();
    if (wave == 0) {
        const int seg = static_cast<int>(sh.pick[0]);
        const int j0 = ((seg / kWaves) * kThreads + seg % kWaves * 64 + lane) * kP;
        u64 m[kP], sum = 0;
        float v[kP];
#pragma unroll
        for (int i = 0; i < kP; ++i) {
            v[i] = j0 + i < R.n ? to_f32(R.x[j0 + i]) : -INFINITY;
            m[i] = j0 + i < R.n ? value(j0 + i, v[i]) : 0;
            sum += m[i];
        }
        before = sh.pick[1] + wave_before(sum);
#pragma unroll
        for (int i = 0; i < kP; ++i) {
            if (m[i] && before <= aim && aim < before + m[i]) found(j0 + i, v[i], total);
            before += m[i];
        }
    }
    __syncthreads();
}

template <class T, int kThreads>
__global__ void __launch_bounds__(kThreads) k_sample(hx_sample_args A) {
    using R_ = Row<T, kThreads>;
    using Sh = Shared<kThreads>;
    constexpr int kP = R_::kP, kBins = Sh::kBins;
    __shared__ Sh sh;
    extern __shared__ u64 segments[];          // sums of each wave's turns in each()
    const long long row = blockIdx.x;
    R_ R;
    R.x = static_cast<const T*>(A.logits) + row * A.logits_stride;
    R.n = static_cast<int>(A.vocab);
    const float temp = A.temperature ? A.temperature[row] : static_cast<float>(A.temperature_value);
    const long long top_k = A.top_k ? A.top_k[row] : A.top_k_value;
    const float top_p = A.top_p ? A.top_p[row] : static_cast<float>(A.top_p_value);
    const float min_p = fminf(A.min_p ? A.min_p[row] : static_cast<float>(A.min_p_value), 1.f);
    const bool greedy = !(temp > 0.f);
    R.cold = greedy ? 1.f : 1.f / temp;
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    if (threadIdx.x == 0) sh.count = 0;

    float most = -INFINITY;                    // fmaxf passes over NaN
    R.each([&](int, const float* v, int) {
#pragma unroll
        for (int i = 0; i < kP; ++i) most = fmaxf(most, v[i]);
    });
    R.most = value_of(block_reduce<kThreads>(key_of(most), sh.part, [](unsigned a, unsigned b) { return max(a, b); }));
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
    if (greedy) {
        int first = R.n;
        R.each([&](int j0, const float* v, int) {
#pragma unroll
            for (int i = 0; i < kP; ++i)
                if (v[i] == R.most) first = min(first, j0 + i);
        });
        first = block_reduce<kThreads>(first, sh.part, [](int a, int b) { return min(a, b); });
        if (threadIdx.x == 0) answer(first, R.most, static_cast<u64>(kMass));
        return;
    }
    auto aim = [&](u64 total) {
        const double u = fmin(fmax(static_cast<double>(A.u[row]), 0.0), 1.0);
        const u64 a = static_cast<u64>(floor(u * static_cast<double>(total)));
        return a < total ? a : total - 1;
    };
    // The largest place stays whatever top_p is.
    auto bound_of = [&](u64 total) { return fmax(static_cast<double>(top_p) * static_cast<double>(total), 0.5); };

    // Places stay whose key is over `least`, and those at it up to index `last`.
    unsigned least = 0;
    int last = R.n;
    auto stays = [&](int j, float v) {
        const unsigned k = key_of(v);
        return k > least || (k == least && j <= last);
    };
    auto last_of = [&](u64 ties) {             // the index of so many places at the key
        at_running_sum(R, sh, segments, [&](int, float v) { return u64(v == v && key_of(v) == least); },
                       [&](u64) { return ties - 1; }, [&](int j, float, u64) { sh.pick[2] = j; });
        last = static_cast<int>(sh.pick[2]);
        __syncthreads();
    };
    if (top_k > 0 && top_k < R.n) {
        auto passes = [&](u64 n) { return n >= static_cast<u64>(top_k); };
        auto one = [](int, float v) { return u64(v == v); };
        add_parts(R, sh, one);
        Cut c = find_bin(sh, passes, 0);
        // (where fewer than top_k places have a mass, all that have one stay)
        u64 mine = kNone;
        bool listed = false;
        if (c.bin >= 0 && c.before + c.at <= kThreads) {
            listed = gather(R, sh, [&](int, float v) { return part_of<kBins>(R, v) >= c.bin; }, mine);
            if (threadIdx.x >= top_k) mine = kNone;
        } else if (c.bin >= 0) {
            least = refine(R, sh, one, passes, c);
            if (top_k - c.before < c.at) last_of(top_k - c.before);
            if (top_k <= kThreads) listed = gather(R, sh, stays, mine);
        }
        if (listed) {
            // in rank order
            const float v = mine != kNone ? ranked_value(mine) : -INFINITY;
            u64 m = mine != kNone ? R.mass(v) : 0, total;
            u64 before = block_before(m, sh, total);
            if (!(top_p >= 1.f) && !(static_cast<double>(before) < bound_of(total))) m = 0;
            if (!(R.weight(v) >= min_p)) m = 0;
            // and in index order
            mine = block_sort<kThreads>(m ? mine << 32 | mine >> 32 : kNone, sh.bins + kThreads);
            const float w = mine != kNone ? value_of(~static_cast<unsigned>(mine)) : -INFINITY;
            m = mine != kNone ? R.mass(w) : 0;
            before = block_before(m, sh, total);
            const u64 to = aim(total);
            if (m && before <= to && to < before + m) answer(static_cast<int>(mine >> 32), w, total);
            return;
        }
    }
    if (!(top_p >= 1.f)) {
        auto counted = [&](int j, float v) { return stays(j, v) ? R.mass(v) : 0; };
        if (least) add_parts(R, sh, counted);
        else add_parts(R, sh, [&](int, float v) { return R.mass(v); });
        __syncthreads();
        u64 total = 0;
        for (int i = threadIdx.x; i < kBins; i += kThreads) total += sh.bins[i];
        const double bound = bound_of(block_sum(total, sh));
        auto passes = [&](u64 s) { return static_cast<double>(s) >= bound; };
        Cut c = find_bin(sh, passes, 0);
        u64 mine;
        if (gather(R, sh, [&](int j, float v) { return part_of<kBins>(R, v) == c.bin && stays(j, v); }, mine)) {
            const u64 m = mine != kNone ? R.mass(ranked_value(mine)) : 0;
            u64 all;
            const u64 before = c.before + block_before(m, sh, all);
            // the last place that stays: less than the bound before it, not after it
            if (m && !passes(before) && passes(before + m)) {
                sh.pick[0] = ~static_cast<unsigned>(mine >> 32);
                sh.pick[1] = static_cast<unsigned>(mine);
            }
            __syncthreads();
            least = static_cast<unsigned>(sh.pick[0]);
            last = static_cast<int>(sh.pick[1]);
            __syncthreads();
        } else {
            const unsigned cut = refine(R, sh, counted, passes, c);
            const u64 m = R.mass(value_of(cut)), at = c.at / m;
            const u64 ties = count_under(bound, c.before, m, at);
            if (cut != least) last = R.n;
            least = cut;
            if (ties < at) last_of(ties);
        }
    }
    at_running_sum(
        R, sh, segments,
        [&](int j, float v) {
            const float w = R.weight(v);
            return stays(j, v) && w >= min_p ? static_cast<u64>(w * kMass) : 0;
        },
        aim, answer);
}

}  // namespace

hipError_t sample_launch(const hx_sample_args& A) {
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto threads) {
            constexpr int kThreads = decltype(threads)::value;
            constexpr int64_t turn = static_cast<int64_t>(kThreads) * Row<T, kThreads>::kP;
            const size_t lds = sizeof(u64) * (kThreads / 64) * ((A.vocab + turn - 1) / turn);
            if (lds > 32768) {
                const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k_sample<T, kThreads>),
                                                         hipFuncAttributeMaxDynamicSharedMemorySize, 140000);
                if (e != hipSuccess) return e;
            }
            k_sample<T, kThreads><<<static_cast<unsigned>(A.rows), kThreads, lds, st>>>(A);
            return hipGetLastError();
        };
        // Threads a row.  A row that has a CU to itself takes 1024 (16000 places: 12 us against 20
        // with 256); small ones and many are faster with 256, whose barriers and sorts are short
        // (1500 rows: of 600 places 24 us against 131, of 16000 places 112 against 176).
        return A.vocab <= 4096 || A.rows >= 1024 ? go(std::integral_constant<int, 256>{})
                                                 : go(std::integral_constant<int, 1024>{});
    });
}

}  // namespace hx
