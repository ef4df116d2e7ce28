// Log probabilities of given tokens with the entropy and the top alternatives of each row of
// logits, and their gradient.
//
// One pass over a row gives z = sum 2^y and s = sum y 2^y, y = (x - base) log2 e / t, from which
// log q = (x - base) / t - ln z and the entropy ln z - ln 2 s / z follow.  The base is the largest
// logit of the row's first pieces; a thread that meets one far above it moves its own.  The top
// places come out of the same pass: every wave's lanes hold the largest logit of their first
// pieces, and a bound that enough of these reach lets few of the row's logits through, a few
// hundred of a hundred thousand.  They wait in LDS as whole numbers, logit above index, and each
// counts those above it.  Where more than 256 come through, the top places' own bound is found
// byte by byte from histograms, of those that came or, where a wave's list is too short for them
// (logits that rise along the row, or are all the same), of the row's values.
//
// Few long rows are cut into parts, which a second launch joins.  Bound by the logits' bytes, read
// once: 2048 x 131072 in bf16 with the top 5 in 106 to 118 us, 4.6 to 5.1 TB/s; short rows by what a
// row starts and ends with.  The gradient reads and writes them once: 1037 x 50021 in fp16 in 40 us, 5.2 TB/s.
#include "readout.h"

#include <algorithm>
#include <type_traits>

namespace hx {
namespace {

typedef unsigned long long u64;

constexpr int kAhead = 4;                  // pieces a thread asks for at a time
constexpr float kFar = 64.f;               // a base is moved where weights pass 2^64
constexpr float kNone = -200.f;            // 2^y is 0 from here on; y = -inf would make y 2^y no number
constexpr double kLn2 = 0.6931471805599453;

struct LogprobArgs {
    const void *logits, *tokens;
    long long stride;
    int vocab, top, index_bits, parts, each;   // each: logits of a part
    float cold;                                // log2 e / temperature
    double per;                                // 1 / temperature
    float *logprob, *entropy, *stats, *top_logprob;
    int64_t* top_index;
    struct Sums* sums;                         // (rows, parts)
    u64* keys;                                 // (rows, parts, top)
};

struct Sums {
    double z, s;
    float base, most;
};

// Logits ordered as whole numbers, above the indexes, lowest first; -0 is 0 and NaN -inf.
__device__ __forceinline__ unsigned order_of(float v) {
    const unsigned b = __float_as_uint(v != v ? -INFINITY : v + 0.f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned o) { return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ u64 key_of(float v, int j) { return static_cast<u64>(order_of(v)) << 32 | ~static_cast<unsigned>(j); }
__device__ __forceinline__ int index_of(u64 key) { return static_cast<int>(~static_cast<unsigned>(key)); }

__device__ __forceinline__ long long token_of(const LogprobArgs& A, long long row) {
    return A.index_bits == 64 ? static_cast<const int64_t*>(A.tokens)[row] : static_cast<const int32_t*>(A.tokens)[row];
}

constexpr int kEach = 544, kBest = 256;    // keys that a wave holds, and that are ranked

// A run of n elements as pieces of 16 bytes that start at multiples of 16, and what is left before and
// after them (rows of 50021 fp16 logits, 1037 of them: 33 us with pieces that start anywhere, 29 so).
template <class T>
struct Pieces {
    static constexpr int kP = 16 / sizeof(T);
    int n, head, count;
    __device__ __forceinline__ Pieces(const T* at, int n) : n(n) {
        head = min(static_cast<int>((16 - reinterpret_cast<uintptr_t>(at) % 16) % 16 / sizeof(T)), n);
        count = (n - head) / kP;
    }
    // the i-th element beside the pieces; n and more: there are not so many
    __device__ __forceinline__ int odd(int i) const { return i < head ? i : i + count * kP; }
};

template <int kThreads>
struct Shared {
    double red[kThreads / 64];
    float most[kThreads / 64], bound[kThreads / 64];
    int count[kThreads / 64], chosen, left;
    unsigned bins[256];
    u64 prefix, answer;
    u64 best[kBest], held[kThreads / 64][kEach];
};

// The k-th largest of a wave's values, to 16 bits of their order (rounded down): at least k of them
// are not below it.
__device__ __forceinline__ float kth_of_wave(float v, int k) {
    const unsigned mine = order_of(v) >> 16;
    unsigned found = 0;
    for (int bit = 15; bit >= 0; --bit) {
        const unsigned tried = found | 1u << bit;
        if (__popcll(__ballot(mine >= tried)) >= k) found = tried;
    }
    return found <= 0x7f ? -INFINITY : value_of(found << 16);
}

// The bound that the `top` largest of `total` keys reach and no others, byte by byte from histograms.
// each(f) calls f(key, whether it is one) for all of them, a whole wave at a time.  Where the bytes
// from kLast bits on do not tell (equal keys) the answer is 0: sh.prefix holds those bytes of the
// last that belong, sh.left how many of them do.
template <int kThreads, int kLast, class Each>
__device__ u64 bound_of(int top, int total, Shared<kThreads>& sh, Each each) {
    const int lane = threadIdx.x % 64;
    if (threadIdx.x == 0) sh.prefix = sh.answer = 0, sh.left = min(top, total);
    for (int shift = 56; shift >= kLast; shift -= 8) {
        for (int b = threadIdx.x; b < 256; b += kThreads) sh.bins[b] = 0;
        __syncthreads();
        const u64 prefix = sh.prefix, answer = sh.answer;
        if (answer) return answer;
        each([&](u64 key, bool is) {
            const bool in = is && (shift == 56 || key >> (shift + 8) == prefix >> (shift + 8));
            const int bin = static_cast<int>(key >> shift & 255);
            const u64 live = __ballot(in);
            if (!live) return;
            const int one = __shfl(bin, __ffsll(live) - 1);
            if (__all(!in || bin == one)) {       // a wave of equal logits adds once
                if (lane == 0) atomicAdd(&sh.bins[one], static_cast<unsigned>(__popcll(live)));
            } else if (in) {
                atomicAdd(&sh.bins[bin], 1u);
            }
        });
        __syncthreads();
        if (threadIdx.x < 64) {
            // a lane for four bins, the highest first: the lane whose bins reach what is left
            int n[4], mine = 0;
            for (int i = 0; i < 4; ++i) mine += n[i] = sh.bins[255 - 4 * lane - i];
            int upto = mine;
            for (int d = 1; d < 64; d *= 2) {
                const int below = __shfl_up(upto, d);
                if (lane >= d) upto += below;
            }
            const int left = sh.left;
            if (upto >= left && upto - mine < left) {
                int rest = left - (upto - mine), i = 0;
                while (n[i] < rest) rest -= n[i++];
                sh.prefix = prefix | static_cast<u64>(255 - 4 * lane - i) << shift;
                sh.left = rest;
                // where the whole bin belongs its first possible key is the bound
                if (n[i] == rest || shift == 0) sh.answer = sh.prefix;
            }
        }
        __syncthreads();
    }
    return sh.answer;
}

// Keys of at least `bound` to sh.best.
template <int kThreads, class Each>
__device__ void choose(u64 bound, Shared<kThreads>& sh, Each each) {
    if (threadIdx.x == 0) sh.chosen = 0;
    __syncthreads();
    each([&](u64 key, bool is) {
        if (is && key >= bound) {
            const int at = atomicAdd(&sh.chosen, 1);
            if (at < kBest) sh.best[at] = key;
        }
    });
    __syncthreads();
}

// Calls put(rank, key) for the top largest of sh.best's keys.
template <int kThreads, class F>
__device__ __forceinline__ void rank_best(int top, const Shared<kThreads>& sh, F put) {
    const int n = min(sh.chosen, kBest);
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 key = sh.best[i];
        int rank = 0;
        for (int k = 0; k < n; ++k) rank += sh.best[k] > key;
        if (rank < top) put(rank, key);
    }
}

// The top largest of a row's n logits from x on, the first of them index `first`, to sh.best: the
// value that bounds them, then all above it and the first of those at it.
template <class T, int kThreads>
__device__ void choose_of_row(const T* x, int n, int first, int top, Shared<kThreads>& sh) {
    using Vec = typename PieceOf<T>::Vec;
    constexpr int kP = sizeof(Vec) / sizeof(T), kWaves = kThreads / 64;
    // the bits of an order that all numbers of the type share
    constexpr int kSame = std::is_same_v<T, float> ? 0 : std::is_same_v<T, __half> ? 8 : 16;
    const int pieces = n / kP, wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int turns = (pieces + kThreads - 1) / kThreads;
    // f(logits, how many, the first one's place) of this thread in a turn; the last turn is what whole pieces leave
    auto turn = [&](int c, auto f) {
        float v[kP];
        const int p = c * kThreads + static_cast<int>(threadIdx.x), j = pieces * kP + static_cast<int>(threadIdx.x);
        int count = 0;
#pragma unroll
        for (int i = 0; i < kP; ++i) v[i] = 0.f;
        if (c == turns) {
            if (j < n) v[0] = to_f32(x[j]), count = 1;
        } else if (p < pieces) {
            const Vec raw = *reinterpret_cast<const Vec*>(x + static_cast<long long>(p) * kP);
#pragma unroll
            for (int i = 0; i < kP; ++i) v[i] = static_cast<float>(raw[i]);
            count = kP;
        }
        f(v, count, c == turns ? j : p * kP);
    };
    const u64 answer = bound_of<kThreads, 32 + kSame>(top, n, sh, [&](auto f) {
        for (int c = 0; c <= turns; ++c)
            turn(c, [&](const float* v, int count, int) {
#pragma unroll
                for (int i = 0; i < kP; ++i) f(static_cast<u64>(order_of(v[i])) << 32, i < count);
            });
    });
    // above `value` all belong, at it the first `left`
    const unsigned value = static_cast<unsigned>((answer ? answer : sh.prefix) >> 32 >> kSame) - (answer ? 1 : 0);
    const int left = answer ? 0 : sh.left, want = min(top, n);
    __syncthreads();
    if (threadIdx.x == 0) sh.chosen = 0;
    __syncthreads();
    auto push = [&](float v, int j) {
        const int at = atomicAdd(&sh.chosen, 1);
        if (at < kBest) sh.best[at] = key_of(v, first + j);
    };
    int before = 0;                               // logits at the bound in earlier turns
    for (int c = 0; c <= turns; ++c) {
        int mine = 0, here = 0;
        turn(c, [&](const float* v, int count, int j) {
#pragma unroll
            for (int i = 0; i < kP; ++i) {
                const unsigned o = order_of(v[i]) >> kSame;
                if (i < count && o > value) push(v[i], j + i);
                mine += i < count && o == value;
            }
            int upto = mine;
            for (int d = 1; d < 64; d *= 2) {
                const int below = __shfl_up(upto, d);
                if (lane >= d) upto += below;
            }
            if (lane == 63) sh.count[wave] = upto;
            __syncthreads();
            int rank = before + upto - mine;
            for (int w = 0; w < kWaves; ++w) {
                here += sh.count[w];
                if (w < wave) rank += sh.count[w];
            }
#pragma unroll
            for (int i = 0; i < kP; ++i)
                if (i < count && order_of(v[i]) >> kSame == value && rank++ < left) push(v[i], j + i);
        });
        before += here;
        __syncthreads();
        const bool done = sh.chosen >= want;      // read by all before the next turn adds to it
        __syncthreads();
        if (done) break;
    }
}

// Calls put(rank, key) for the top largest keys, from the largest on, of the waves' lists or, where one
// was too short, of the n logits from x on.
template <class T, int kThreads, class F>
__device__ __forceinline__ void each_ranked(const T* x, int n, int first, int top, Shared<kThreads>& sh, F put) {
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    int total = 0, longest = 0;
    for (int v = 0; v < kThreads / 64; ++v) {
        total += sh.count[v];
        longest = max(longest, sh.count[v]);
    }
    auto held = [&](auto f) {
        for (int i = 0; i < sh.count[wave]; i += 64) f(i + lane < sh.count[wave] ? sh.held[wave][i + lane] : 0, i + lane < sh.count[wave]);
    };
    __syncthreads();
    if (longest > kEach) choose_of_row<T, kThreads>(x, n, first, top, sh);
    else choose<kThreads>(total > kBest ? bound_of<kThreads, 0>(top, total, sh, held) : 0, sh, held);
    rank_best<kThreads>(top, sh, put);
}

// A row's results from its sums.  Every thread has the same sums; keys go through put_top.
struct Finish {
    double logz;
    float base, most;
    bool none, broken;                        // nothing but -inf; NaN or +inf among the logits
    __device__ __forceinline__ Finish(const Sums& S) : logz(log(S.z)), base(S.base), most(S.most) {
        broken = !(S.z < INFINITY) || S.most == INFINITY;
        none = !broken && S.most == -INFINITY;
    }
    __device__ __forceinline__ float logprob(float v, double per) const {
        if (broken) return NAN;
        return v == -INFINITY ? -INFINITY : static_cast<float>((static_cast<double>(v) - base) * per - logz);
    }
};

template <class T>
__device__ __forceinline__ void finish_row(const LogprobArgs& A, long long row, const T* x, const Sums& S, const Finish& f) {
    const long long token = token_of(A, row);
    A.logprob[row] = token < 0 || token >= A.vocab ? 0.f : f.logprob(to_f32(x[token]), A.per);
    A.entropy[row] = f.broken ? NAN : f.none ? 0.f : static_cast<float>(fmax(f.logz - kLn2 * S.s / S.z, 0.));
    A.stats[2 * row] = f.broken ? NAN : f.most;
    A.stats[2 * row + 1] = f.broken ? NAN : f.none ? -INFINITY
                                                  : static_cast<float>(f.logz + (static_cast<double>(f.base) - f.most) * A.per);
}

__device__ __forceinline__ void put_top(const LogprobArgs& A, long long row, const Finish& f, int rank, u64 key) {
    A.top_index[row * A.top + rank] = index_of(key);
    A.top_logprob[row * A.top + rank] = f.logprob(value_of(static_cast<unsigned>(key >> 32)), A.per);
}

// One workgroup a part of a row (the whole row, where it is not cut).
template <class T, int kThreads, bool kTop>
__global__ void __launch_bounds__(kThreads, 8) k_logprobs(LogprobArgs A) {
    using Vec = typename PieceOf<T>::Vec;
    constexpr int kP = sizeof(Vec) / sizeof(T), kWaves = kThreads / 64;
    __shared__ Shared<kThreads> sh;
    const long long row = blockIdx.x / A.parts;
    const int part = static_cast<int>(blockIdx.x - row * A.parts);
    const T* x = static_cast<const T*>(A.logits) + row * A.stride;
    const int first = part * A.each, last = min(first + A.each, A.vocab);
    const Pieces<T> cut(x + first, last - first);
    const int pieces = cut.count;
    const T* from = x + first + cut.head;
    Vec raw[kAhead];
    auto fetch = [&](int p0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (p0 + k * kThreads < pieces)
                raw[k] = *reinterpret_cast<const Vec*>(from + static_cast<long long>(p0 + k * kThreads) * kP);
    };
    fetch(threadIdx.x);
    // the logits that are left beside whole pieces, one a thread
    const int odd = first + cut.odd(threadIdx.x);
    const bool has_odd = odd < last;
    const float one = has_odd ? to_f32(x[odd]) : -INFINITY;

    float most = has_odd ? fmaxf(one, -INFINITY) : -INFINITY;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (static_cast<int>(threadIdx.x) + k * kThreads < pieces)
#pragma unroll
            for (int i = 0; i < kP; ++i) most = fmaxf(most, static_cast<float>(raw[k][i]));
    float bound = -INFINITY;
    {
        const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
        // Waves whose every lane holds a piece share the top places among them: `quota` of a wave's
        // lanes are not below its own bound, and the bound that `need` waves reach holds for all.
        const int full = min(pieces, kThreads) / 64, quota = full ? max(1, (A.top + full - 1) / full) : 65;
        const int need = (A.top + quota - 1) / quota;
        float m = most;
        for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        if (kTop && quota <= 64) bound = quota == 1 ? m : kth_of_wave(most, quota);
        if (lane == 0) sh.most[wave] = m, sh.bound[wave] = wave < full ? bound : -INFINITY;
        __syncthreads();
        const float mine = lane < kWaves ? sh.bound[lane] : -INFINITY;
        int above = 0;
        for (int v = 0; v < kWaves; ++v) {
            most = fmaxf(most, sh.most[v]);
            const float other = sh.bound[v];
            above += other > mine || (other == mine && v < lane);
        }
        if (kTop && quota <= 64) bound = __shfl(mine, __ffsll(__ballot(lane < kWaves && above == need - 1)) - 1);
    }
    float base = most == -INFINITY ? 0.f : most, limit = most == -INFINITY ? -INFINITY : base + kFar / A.cold;
    // z and s of kAhead pieces in fp32, at most 8 terms and 4 pieces added one after another, of all in 64 bits:
    // a thread of a long row adds thousands of terms, and where these are alike their roundings are too.
    float z = 0.f, s = 0.f;
    double all_z = 0., all_s = 0.;
    auto fold = [&] {
        all_z += z;
        all_s += s;
        z = s = 0.f;
    };
    // A wave's own list: no atomics, and no wait before the next logits.  The lanes that call are a
    // wave's first ones, so that lane 0 has counted them all.
    int kept = 0;
    auto keep = [&](float v, int j) {
        const bool in = (v != v ? -INFINITY : v) >= bound;
        const u64 those = __ballot(in);
        if (!those) return;
        const int before = __builtin_amdgcn_readfirstlane(kept);
        const int at = before + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(those >> 32),
                                                        __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(those), 0));
        if (in && at < kEach) sh.held[threadIdx.x / 64][at] = key_of(v, j);
        kept = before + __popcll(those);
    };
    auto take = [&](const float* v, int n, int j) {
        float c = v[0];
#pragma unroll
        for (int i = 1; i < kP; ++i)
            if (i < n) c = fmaxf(c, v[i]);
        most = fmaxf(most, c);
        if (c > limit) {
            fold();
            const float less = all_z == 0. ? 0.f : fmaxf((base - c) * A.cold, -1e9f);
            const double f = __builtin_amdgcn_exp2f(less);
            all_s = f * (all_s + less * all_z);
            all_z *= f;
            base = c;
            limit = c + kFar / A.cold;
        }
        float piece_z = 0.f, piece_s = 0.f;
#pragma unroll
        for (int i = 0; i < kP; ++i)
            if (i < n) {
                const float y = (v[i] - base) * A.cold, w = __builtin_amdgcn_exp2f(y);
                piece_z += w;
                piece_s = fmaf(w, fmaxf(y, kNone), piece_s);
            }
        z += piece_z;
        s += piece_s;
        if constexpr (kTop)
            if (__any(!(c < bound)))
#pragma unroll
                for (int i = 0; i < kP; ++i)
                    if (i < n) keep(v[i], j + i);
    };
    for (int p0 = threadIdx.x; p0 < pieces; p0 += kAhead * kThreads) {
        if (p0 != static_cast<int>(threadIdx.x)) fetch(p0);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int p = p0 + k * kThreads;
            if (p < pieces) {
                float v[kP];
#pragma unroll
                for (int i = 0; i < kP; ++i) v[i] = static_cast<float>(raw[k][i]);
                take(v, kP, first + cut.head + p * kP);
            }
        }
        fold();
    }
    if (has_odd) {
        const float v[kP] = {one};
        take(v, 1, odd);
        fold();
    }
    // one base for the workgroup: the highest
    const float mine = base;
    auto up = [](float a, float b) { return fmaxf(a, b); };
    auto add = [](double a, double b) { return a + b; };
    Sums S;
    S.most = block_reduce<kThreads>(most, sh.most, up);
    S.base = block_reduce<kThreads>(all_z == 0. ? -INFINITY : base, sh.bound, up);
    if (S.base == -INFINITY) S.base = 0.f;
    const double less = (static_cast<double>(mine) - S.base) * A.cold;
    const double f = mine == S.base || all_z == 0. ? 1. : static_cast<double>(__builtin_amdgcn_exp2f(static_cast<float>(less)));
    S.s = block_reduce<kThreads>(f * (all_s + (all_z == 0. ? 0. : less * all_z)), sh.red, add);
    S.z = block_reduce<kThreads>(f * all_z, sh.red, add);
    if constexpr (kTop) {
        if (threadIdx.x % 64 == 0) sh.count[threadIdx.x / 64] = kept;
        __syncthreads();
    }
    if (A.parts == 1) {
        const Finish done(S);
        if (threadIdx.x == 0) finish_row(A, row, x, S, done);
        if constexpr (kTop)
            each_ranked<T, kThreads>(x + first, last - first, first, A.top, sh, [&](int rank, u64 key) { put_top(A, row, done, rank, key); });
    } else {
        if (threadIdx.x == 0) A.sums[blockIdx.x] = S;
        if constexpr (kTop) {
            u64* const to = A.keys + static_cast<long long>(blockIdx.x) * A.top;
            for (int i = last - first + threadIdx.x; i < A.top; i += kThreads) to[i] = 0;
            each_ranked<T, kThreads>(x + first, last - first, first, A.top, sh, [&](int rank, u64 key) { to[rank] = key; });
        }
    }
}

// The parts of a row, joined.
template <class T>
__global__ void __launch_bounds__(256) k_logprob_join(LogprobArgs A) {
    __shared__ Shared<256> sh;
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(A.logits) + row * A.stride;
    Sums S{0., 0., -INFINITY, -INFINITY};
    for (int p = 0; p < A.parts; ++p) {
        const Sums P = A.sums[row * A.parts + p];
        S.most = fmaxf(S.most, P.most);
        if (P.z != 0.) S.base = fmaxf(S.base, P.base);
    }
    if (S.base == -INFINITY) S.base = 0.f;
    for (int p = 0; p < A.parts; ++p) {
        const Sums P = A.sums[row * A.parts + p];
        const double less = P.z == 0. ? 0. : (static_cast<double>(P.base) - S.base) * A.cold, f = exp2(less);
        S.z += f * P.z;
        S.s += f * (P.s + less * P.z);
    }
    const Finish done(S);
    if (threadIdx.x == 0) finish_row(A, row, x, S, done);
    const int n = A.parts * A.top;
    auto all = [&](auto f) {
        for (int i0 = 0; i0 < n; i0 += 256) {
            const int i = i0 + static_cast<int>(threadIdx.x);
            const u64 key = i < n ? A.keys[row * n + i] : 0;
            f(key, key != 0);
        }
    };
    if (!A.top) return;
    choose<256>(n > kBest ? bound_of<256, 0>(A.top, n, sh, all) : 0, sh, all);
    rank_best<256>(A.top, sh, [&](int rank, u64 key) { put_top(A, row, done, rank, key); });
}

struct GradArgs {
    const void *logits, *tokens;
    void* grad;
    long long rows, stride, grad_stride;
    int vocab, index_bits, blocks;
    float cold, per;
    const float *stats, *entropy, *pull, *turn;
};

// The gradient, kAhead pieces a thread.
template <class T, int kThreads>
__global__ void __launch_bounds__(kThreads) k_logprob_grad(GradArgs A) {
    using Vec = typename PieceOf<T>::Vec;
    constexpr int kP = sizeof(Vec) / sizeof(T);
    for (long long id = blockIdx.x; id < A.rows * A.blocks; id += gridDim.x) {
        const long long row = id / A.blocks;
        const int block = static_cast<int>(id - row * A.blocks);
        const T* x = static_cast<const T*>(A.logits) + row * A.stride;
        T* g = static_cast<T*>(A.grad) + row * A.grad_stride;
        const Pieces<T> cut(g, A.vocab);
        const int pieces = cut.count, p0 = block * kAhead * kThreads + threadIdx.x;
        Vec raw[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (p0 + k * kThreads < pieces)
                raw[k] = *reinterpret_cast<const Vec*>(x + cut.head + static_cast<long long>(p0 + k * kThreads) * kP);
        const long long named = A.index_bits == 64 ? static_cast<const int64_t*>(A.tokens)[row]
                                                   : static_cast<const int32_t*>(A.tokens)[row];
        const int token = named >= 0 && named < A.vocab ? static_cast<int>(named) : -1;
        const float most = A.stats[2 * row], logz2 = A.stats[2 * row + 1] * 1.44269504088896341f;
        const float pull = token >= 0 && A.pull ? A.pull[row] * A.per : 0.f, turn = A.turn ? A.turn[row] * A.per : 0.f;
        const bool none = most == -INFINITY;
        // q (a + b log2 q)
        const float a = -(pull + turn * A.entropy[row]), b = -turn * static_cast<float>(kLn2);
        auto slope = [&](float v) {
            const float l = (v - most) * A.cold - logz2;
            return none ? 0.f : __builtin_amdgcn_exp2f(l) * fmaf(b, fmaxf(l, kNone), a);
        };
        // at the token pull (1 - q), not a difference of nearly equal numbers
        auto slope_at_token = [&](float v) {
            const float l = (v - most) * A.cold - logz2;
            const float r = __builtin_amdgcn_exp2f(l) * fmaf(b, fmaxf(l, kNone), a + pull);
            return none ? 0.f : fmaf(-pull, expm1f(l * static_cast<float>(kLn2)), r);
        };
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int p = p0 + k * kThreads;
            if (p < pieces) {
                Vec out;
                auto put = [&](int i, float r) { out[i] = static_cast<decltype(out[0] + out[0])>(r); };
#pragma unroll
                for (int i = 0; i < kP; ++i) put(i, slope(static_cast<float>(raw[k][i])));
                const int mine = token - cut.head - p * kP;      // the token's place in the piece
                if (mine >= 0 && mine < kP) {
                    float v = 0.f;
#pragma unroll
                    for (int i = 0; i < kP; ++i) v = mine == i ? static_cast<float>(raw[k][i]) : v;
                    const float r = slope_at_token(v);
#pragma unroll
                    for (int i = 0; i < kP; ++i)
                        if (mine == i) put(i, r);
                }
                *reinterpret_cast<Vec*>(g + cut.head + static_cast<long long>(p) * kP) = out;
            }
        }
        const int odd = cut.odd(threadIdx.x);
        if (block == 0 && odd < A.vocab) {
            const float v = to_f32(x[odd]);
            g[odd] = from_f32<T>(odd == token ? slope_at_token(v) : slope(v));
        }
    }
}

// Parts of a row: one, but where rows alone leave CUs without work; of 16384 logits and more each
// (1 x 262144 in bf16: 48 us whole, 21 in parts, 25 in parts of 8192; 300 x 131072: 47 and 37).
int parts_of(const hx_logprob_args& A) {
    if (A.rows >= 512) return 1;
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({1024 / A.rows, A.vocab / 16384, 64})));
}

}  // namespace

size_t logprob_workspace(const hx_logprob_args& A) {
    const int parts = parts_of(A);
    return parts > 1 ? A.rows * parts * (sizeof(Sums) + sizeof(u64) * A.top) : 0;
}

hipError_t logprob_launch(const hx_logprob_args& A) {
    LogprobArgs L{};
    L.logits = A.logits, L.tokens = A.tokens, L.stride = A.logits_stride;
    L.vocab = static_cast<int>(A.vocab), L.top = static_cast<int>(A.top), L.index_bits = static_cast<int>(A.index_bits);
    L.cold = static_cast<float>(1.4426950408889634 / A.temperature), L.per = 1.0 / A.temperature;
    L.logprob = A.logprob, L.entropy = A.entropy, L.stats = A.stats;
    L.top_logprob = A.top_logprob, L.top_index = A.top_index;
    L.parts = parts_of(A);
    L.each = ((L.vocab + L.parts - 1) / L.parts + 7) / 8 * 8;
    L.sums = static_cast<Sums*>(A.workspace);
    L.keys = reinterpret_cast<u64*>(L.sums + A.rows * L.parts);
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    return with_type(A.type, [&](auto t) -> hipError_t {
        using T = decltype(t);
        const unsigned grid = static_cast<unsigned>(A.rows * L.parts);
        auto go = [&](auto threads, auto top) {
            constexpr int kThreads = decltype(threads)::value;
            k_logprobs<T, kThreads, decltype(top)::value><<<grid, kThreads, 0, st>>>(L);
        };
        // Threads: 512 keep four rows on a CU, whose starts and ends lie beside the others' middles (2048 x
        // 131072 in bf16, top 5: 118 us, with 1024 threads 127, with 256 143; top 100: 176 and 188); of
        // short rows 256 threads keep eight (4000 x 32000 in fp16, top 20: 83 us, with 512 threads 88; 300
        // of them, that do not fill the chip, 25 and 19).  More
        // than 128 top places would pass more logits to each of eight waves than its list holds (top
        // 256: 232 us with 1024 threads, 997 with 512).
        auto pick = [&](auto with_top) {
            if (L.each <= 512) go(std::integral_constant<int, 64>{}, with_top);
            else if (L.each <= (grid >= 1024 ? 32768 : 8192)) go(std::integral_constant<int, 256>{}, with_top);
            else if (A.top <= 128) go(std::integral_constant<int, 512>{}, with_top);
            else if constexpr (decltype(with_top)::value) go(std::integral_constant<int, 1024>{}, with_top);
        };
        A.top ? pick(std::true_type{}) : pick(std::false_type{});
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || L.parts == 1) return e;
        k_logprob_join<T><<<static_cast<unsigned>(A.rows), 256, 0, st>>>(L);
        return hipGetLastError();
    });
}

hipError_t logprob_gradient(const hx_logprob_args& A) {
    GradArgs G{};
    G.logits = A.logits, G.tokens = A.tokens, G.grad = A.grad;
    G.rows = A.rows, G.stride = A.logits_stride, G.grad_stride = A.grad_stride;
    G.vocab = static_cast<int>(A.vocab), G.index_bits = static_cast<int>(A.index_bits);
    G.cold = static_cast<float>(1.4426950408889634 / A.temperature), G.per = static_cast<float>(1.0 / A.temperature);
    G.stats = A.stats, G.entropy = A.entropy, G.pull = A.grad_logprob, G.turn = A.grad_entropy;
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto threads) {
            constexpr int kThreads = decltype(threads)::value, kTurn = kThreads * kAhead * static_cast<int>(16 / sizeof(T));
            G.blocks = (G.vocab + kTurn - 1) / kTurn;
            const unsigned grid = static_cast<unsigned>(std::min<long long>(A.rows * G.blocks, 1 << 23));
            k_logprob_grad<T, kThreads><<<grid, kThreads, 0, static_cast<hipStream_t>(A.stream)>>>(G);
        };
        if (G.vocab <= 1024) go(std::integral_constant<int, 64>{});
        else go(std::integral_constant<int, 256>{});
        return hipGetLastError();
    });
}

}  // namespace hx
