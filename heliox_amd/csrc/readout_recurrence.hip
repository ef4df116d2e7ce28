// A gated recurrence for each channel, h_t = (1 - z_t) h_{t-1} + z_t x_t, z = 1 / (1 + e^gate), and
// its gradient.
//
// A run of steps takes what enters it to P h + Y (P the product of the a = 1 - z, Y what the run
// makes of nothing), and runs join: that is the scan.  What is left of P and h is h - z h in one
// rounding, not a h: a channel that remembers for a thousand steps has a = 0.999, whose last bit
// counts a thousand times, while z keeps all of its bits.  Where the gate shuts it is the other way
// round: there z is nearly 1, and a h with a = e^gate z has the bits.
//
// Lanes lie along channels, kC each, so that a step's row is read and written as it lies in
// memory; a group of kL lanes (a wave; fewer, where there are few channels) takes kU steps in
// registers, a workgroup's groups take as many more in a row and join in LDS.  Where sequences
// and channels alone fill the chip a workgroup walks along its whole sequence, one pass over the
// data.  Where they do not, sequences are cut into segments: one launch makes each segment's P
// and Y, one joins them, one walks the segments.  The gradient goes that way always, a segment
// being a workgroup's steps: what the future hands back to a run, G = R + P G', joins from the
// right as h does from the left, and both meet in the run's registers.
//
// Bound by memory, at 4.4 to 5.2 TB/s of what the passes move (a copy: 4.9): 8 x 4096 x 2048 in bf16
// forward 89 us (402 MB once), backward 217 (1074 MB: inputs twice); 65536 x 512 in fp32 forward,
// cut, 135 us (671 MB).
#include "readout.h"

#include <algorithm>
#include <type_traits>

namespace hx {
namespace {

constexpr int kThreads = 512;
template <int kC> constexpr int kU = 16 / kC;                              // steps that a lane holds
template <int kC, int kL> constexpr int kTile = kU<kC> * (kThreads / kL);  // and a workgroup

struct RecurrenceArgs {
    const void *x, *gate, *grad_o;
    long long x_stride[2], gate_stride[2], grad_o_stride[2], o_stride[2];
    void *o, *grad_x, *grad_gate;
    const int32_t* lengths;
    const float *initial, *grad_end;
    float *end, *grad_initial;
    float *p, *y, *r;                // (batch, segments, channels): P, Y and R of each segment
    float *enter, *leave;            // the same: what enters it from the left and, going back, from the right
    int time, channels, blocks;      // blocks: of kL kC channels
    int segments, steps;             // steps: of a segment
    long long batch;
    bool runs;                       // how places are dealt out: see each_place
};

template <class T, int kC> struct Packed;
template <> struct Packed<float, 1> { typedef float Vec; };
template <> struct Packed<__half, 2> { typedef _Float16 Vec __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Packed<__hip_bfloat16, 2> { typedef __bf16 Vec __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Packed<__half, 1> { typedef _Float16 Vec; };
template <> struct Packed<__hip_bfloat16, 1> { typedef __bf16 Vec; };

template <class Vec, int kC>
__device__ __forceinline__ float part(const Vec& v, int c) {
    if constexpr (kC == 1) return static_cast<float>(v);
    else return static_cast<float>(v[c]);
}

template <class T, int kC>
__device__ __forceinline__ typename Packed<T, kC>::Vec packed(const float* x) {
    typename Packed<T, kC>::Vec v;
    if constexpr (kC == 1) {
        v = static_cast<typename Packed<T, kC>::Vec>(x[0]);
    } else {
#pragma unroll
        for (int c = 0; c < kC; ++c) v[c] = static_cast<decltype(v[0] + v[0])>(x[c]);
    }
    return v;
}

// e^gate; infinite over 88.
__device__ __forceinline__ float rise(float gate) { return __builtin_amdgcn_exp2f(gate * 1.44269504088896341f); }
// 1 / (1 + e^gate) from e^gate
__device__ __forceinline__ float opening(float e) { return __builtin_amdgcn_rcpf(1.f + e); }

// Gates up to here shut: at -1 z = 0.73 is off by at most 4 halves of a step, a = 1 - z by 10 of its own, as
// e^gate z is there.  (Of e^gate the exponent's rounding is the most, 22 halves at -25.)
constexpr float kShut = -1.f;

// A step's opening z and what it keeps, a.  Waves whose steps do not shut (kShuts false: see any_shuts)
// go without what that takes, with the same results: 8 x 4096 x 2048 with gradient 313 us, with it
// everywhere 321, where steps shut in every wave 317.
template <bool kShuts>
struct Opening {
    float z, a;
    bool shut;
    __device__ __forceinline__ Opening() {}
    __device__ __forceinline__ Opening(float gate, bool live) {
        const float e = rise(gate);
        z = live ? opening(e) : 0.f;
        a = !live || gate > 80.f ? 1.f : e * z;
        shut = kShuts && live && gate <= kShut;
    }
    // what is left of h, and h moved towards x
    __device__ __forceinline__ float left(float h) const { return fmaf(shut ? a : -z, h, shut ? 0.f : h); }
    __device__ __forceinline__ float moved(float h, float x) const { return fmaf(z, x, left(h)); }
};

// Whether some of the wave's gates are kShut or less: of the numbers' bits, as whole numbers without a
// sign, those of negative ones are the largest, the more so the further from zero.
template <int kC, class Vec, int kN>
__device__ __forceinline__ bool any_shuts(const Vec (&gates)[kN]) {
    unsigned most = 0;
#pragma unroll
    for (int u = 0; u < kN; ++u)
#pragma unroll
        for (int c = 0; c < kC; ++c) most = max(most, __float_as_uint(part<Vec, kC>(gates[u], c)));
    return __any(most >= __float_as_uint(kShut));
}

// Calls f(whether all steps are within the length, whether some shut).
template <class F>
__device__ __forceinline__ void with_kind(bool whole, bool shuts, F f) {
    if (!whole) f(std::false_type{}, std::true_type{});
    else if (shuts) f(std::true_type{}, std::true_type{});
    else f(std::true_type{}, std::false_type{});
}

// A workgroup's place: sequence, segment, channels.
struct Where {
    long long batch;
    int segment, channel, length;
    template <int kC, int kL>
    __device__ __forceinline__ static Where of(const RecurrenceArgs& A, long long id) {
        Where w;
        const long long row = id / A.blocks;
        // lanes past the last channel do the last channels over again, and write the same values
        w.channel = min((static_cast<int>(id - row * A.blocks) * kL + static_cast<int>(threadIdx.x) % kL) * kC,
                        A.channels - kC);
        w.batch = row / A.segments;
        w.segment = static_cast<int>(row - w.batch * A.segments);
        w.length = A.lengths ? min(max(A.lengths[w.batch], 0), A.time) : A.time;
        return w;
    }
    __device__ __forceinline__ long long at(const RecurrenceArgs& A) const { return at(A, segment); }
    __device__ __forceinline__ long long at(const RecurrenceArgs& A, int s) const {
        return (batch * A.segments + s) * A.channels + channel;
    }
    // What enters the segment from the left, and going back from the right: as it was joined, or, with
    // kJoins, what enters the sequence, taken along the segments beside this one.  (Variants of their
    // own: with both ways in one kernel its loads wait for each other, 306 us for 8 x 4096 x 2048
    // with gradient became 309 to 317.)
    template <bool kJoins, int kC>
    __device__ __forceinline__ void entering(const RecurrenceArgs& A, float (&h)[kC]) const {
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            h[c] = 0.f;
            if (!kJoins && A.segments > 1) h[c] = A.enter[at(A) + c];
            else if (A.initial) h[c] = A.initial[batch * A.channels + channel + c];
        }
        if constexpr (kJoins)
#pragma unroll 8
            for (int s = 0; s < segment; ++s)
#pragma unroll
                for (int c = 0; c < kC; ++c) h[c] = fmaf(A.p[at(A, s) + c], h[c], A.y[at(A, s) + c]);
    }
    template <bool kJoins, int kC>
    __device__ __forceinline__ void leaving(const RecurrenceArgs& A, float (&g)[kC]) const {
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            g[c] = 0.f;
            if (!kJoins && A.segments > 1) g[c] = A.leave[at(A) + c];
            else if (A.grad_end) g[c] = A.grad_end[batch * A.channels + channel + c];
        }
        if constexpr (kJoins)
#pragma unroll 8
            for (int s = A.segments - 1; s > segment; --s)
#pragma unroll
                for (int c = 0; c < kC; ++c) g[c] = fmaf(A.p[at(A, s) + c], g[c], A.r[at(A, s) + c]);
    }
};

// Calls f for this workgroup's share of all places.  Workgroups go to the eight XCDs in turn, and each
// XCD has a cache of its own.  In runs an XCD gets places side by side, so that lines which two
// neighbouring blocks of channels share are read once: for rows that do not start at lines (4 x
// 5500 x 926 in bf16, with gradient: 127 us, in turn 155; 8 x 4096 x 2048, whose rows do: 315 and 306).
template <class F>
__device__ __forceinline__ void each_place(const RecurrenceArgs& A, F f) {
    const long long n = A.batch * A.segments * A.blocks, share = (n + 7) / 8;
    for (long long k = blockIdx.x; k < share * 8; k += gridDim.x) {
        const long long place = A.runs ? k % 8 * share + k / 8 : k;
        if (place < n) f(place);
    }
}

// Which of a workgroup's kThreads / kL groups of lanes this is.
template <int kL>
__device__ __forceinline__ int group_of() {
    const int group = threadIdx.x / kL;
    return kL == 64 ? __builtin_amdgcn_readfirstlane(group) : group;
}

// kU steps from t on of one array; steps past the length are not read.
template <class T, int kC, int kN>
__device__ __forceinline__ void fetch(typename Packed<T, kC>::Vec (&to)[kN], const void* base, const long long (&stride)[2],
                                      const Where& w, int t) {
    using Vec = typename Packed<T, kC>::Vec;
    const T* at = static_cast<const T*>(base) + w.batch * stride[0] + t * stride[1];
    if (t + kN <= w.length) {
#pragma unroll
        for (int u = 0; u < kN; ++u, at += stride[1]) to[u] = *reinterpret_cast<const Vec*>(at + w.channel);
    } else {
#pragma unroll
        for (int u = 0; u < kN; ++u, at += stride[1])
            to[u] = t + u < w.length ? *reinterpret_cast<const Vec*>(at + w.channel) : Vec{};
    }
}

// The whole walk.
template <class T, int kC, int kL, bool kJoins>
__global__ void __launch_bounds__(kThreads, kL == 64 ? 4 : 2) k_walk(RecurrenceArgs A) {
    constexpr int kU = hx::kU<kC>, kTile = hx::kTile<kC, kL>, kW = kThreads / kL;
    using Vec = typename Packed<T, kC>::Vec;
    __shared__ float ends[2][kW][2 * kC][kL];
    const int group = group_of<kL>(), lane = threadIdx.x % kL;
    int turn = 0;
    // (the segments' own launch went over the data from its start: its end is in the cache)
    each_place(A, [&](long long place) {
        const long long id = A.batch * A.segments * A.blocks - 1 - place;
        const Where w = Where::of<kC, kL>(A, id);
        const int first = w.segment * A.steps, last = min(first + A.steps, A.time);
        float h[kC];
        w.entering<kJoins>(A, h);
        Vec x[kU], g[kU];
        fetch<T, kC>(x, A.x, A.x_stride, w, first + group * kU);
        fetch<T, kC>(g, A.gate, A.gate_stride, w, first + group * kU);
        for (int tile = first; tile < last; tile += kTile, turn ^= 1) {
            const int t = tile + group * kU;
            float p[kU][kC], y[kU][kC];
            auto run = [&](auto whole, auto shuts) {
                float pp[kC], yy[kC];
#pragma unroll
                for (int c = 0; c < kC; ++c) pp[c] = 1.f, yy[c] = 0.f;
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    const bool live = decltype(whole)::value || t + u < w.length;
#pragma unroll
                    for (int c = 0; c < kC; ++c) {
                        const Opening<decltype(shuts)::value> open(part<Vec, kC>(g[u], c), live);
                        const float v = live ? part<Vec, kC>(x[u], c) : 0.f;
                        p[u][c] = pp[c] = open.left(pp[c]);
                        y[u][c] = yy[c] = open.moved(yy[c], v);
                    }
                }
            };
            // With one channel a lane asking after the run, which is done over where steps shut, keeps the
            // loads' order (8 x 4096 x 2048: 91 us, asking first 101; two channels, 13 x 777 x 601: 13.1 and 12.1).
            if (kC == 1 && t + kU <= w.length) {
                run(std::true_type{}, std::false_type{});
                if (any_shuts<kC>(g)) run(std::true_type{}, std::true_type{});
            } else {
                with_kind(t + kU <= w.length, any_shuts<kC>(g), run);
            }
            if (tile + kTile < last) {
                fetch<T, kC>(x, A.x, A.x_stride, w, t + kTile);
                fetch<T, kC>(g, A.gate, A.gate_stride, w, t + kTile);
            }
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                ends[turn][group][c][lane] = p[kU - 1][c];
                ends[turn][group][kC + c][lane] = y[kU - 1][c];
            }
            __syncthreads();
            float mine[kC];
#pragma unroll
            for (int c = 0; c < kC; ++c) mine[c] = h[c];
#pragma unroll 8
            for (int v = 0; v < kW; ++v)
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    if (v == group) mine[c] = h[c];
                    h[c] = fmaf(ends[turn][v][c][lane], h[c], ends[turn][v][kC + c][lane]);
                }
            T* o = static_cast<T*>(A.o) + w.batch * A.o_stride[0] + t * A.o_stride[1];
            auto write = [&](auto whole) {
#pragma unroll
                for (int u = 0; u < kU; ++u, o += A.o_stride[1]) {
                    float out[kC];
#pragma unroll
                    for (int c = 0; c < kC; ++c) {
                        const float v = fmaf(p[u][c], mine[c], y[u][c]);
                        out[c] = decltype(whole)::value || t + u < w.length ? v : 0.f;
                    }
                    if (decltype(whole)::value || t + u < A.time)
                        *reinterpret_cast<Vec*>(o + w.channel) = packed<T, kC>(out);
                }
            };
            if (t + kU <= w.length) write(std::true_type{});
            else write(std::false_type{});
        }
        if (A.end && w.segment == A.segments - 1 && group == 0)
#pragma unroll
            for (int c = 0; c < kC; ++c) A.end[w.batch * A.channels + w.channel + c] = h[c];
    });
}

// P, Y (and, for the gradient, R) of each segment: every wave takes a share of its steps.
template <class T, int kC, int kL, bool kGrad>
__global__ void __launch_bounds__(kThreads, kL == 64 ? 4 : 2) k_segments(RecurrenceArgs A) {
    constexpr int kU = hx::kU<kC>, kW = kThreads / kL;
    using Vec = typename Packed<T, kC>::Vec;
    constexpr int kN = kGrad ? 3 : 2;
    __shared__ float ends[kW][kN * kC][kL];
    const int group = group_of<kL>(), lane = threadIdx.x % kL;
    each_place(A, [&](long long id) {
        const Where w = Where::of<kC, kL>(A, id);
        const int each = A.steps / kW, first = w.segment * A.steps + group * each;
        const int last = min(first + each, w.length);
        float p[kC], y[kC], r[kC];
#pragma unroll
        for (int c = 0; c < kC; ++c) p[c] = 1.f, y[c] = r[c] = 0.f;
        for (int t = first; t < last; t += kU) {
            Vec x[kU], g[kU], d[kU];
            fetch<T, kC>(x, A.x, A.x_stride, w, t);
            fetch<T, kC>(g, A.gate, A.gate_stride, w, t);
            if constexpr (kGrad) fetch<T, kC>(d, A.grad_o, A.grad_o_stride, w, t);
            auto run = [&](auto whole, auto shuts) {
#pragma unroll
                for (int u = 0; u < kU; ++u)
                    if (decltype(whole)::value || t + u < last)
#pragma unroll
                        for (int c = 0; c < kC; ++c) {
                            const Opening<decltype(shuts)::value> open(part<Vec, kC>(g[u], c), true);
                            p[c] = open.left(p[c]);
                            y[c] = open.moved(y[c], part<Vec, kC>(x[u], c));
                            if constexpr (kGrad) r[c] = fmaf(p[c], part<Vec, kC>(d[u], c), r[c]);
                        }
            };
            with_kind(t + kU <= last, any_shuts<kC>(g), run);
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            ends[group][c][lane] = p[c];
            ends[group][kC + c][lane] = y[c];
            if constexpr (kGrad) ends[group][2 * kC + c][lane] = r[c];
        }
        __syncthreads();
        if (group == 0)
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                float pp = p[c], yy = y[c], rr = r[c];
#pragma unroll 8
                for (int v = 1; v < kW; ++v) {
                    const float q = ends[v][c][lane];
                    yy = fmaf(q, yy, ends[v][kC + c][lane]);
                    if constexpr (kGrad) rr = fmaf(pp, ends[v][2 * kC + c][lane], rr);
                    pp *= q;
                }
                A.p[w.at(A) + c] = pp;
                A.y[w.at(A) + c] = yy;
                if constexpr (kGrad) A.r[w.at(A) + c] = rr;
            }
    });
}

// What enters each segment from the left, and going back from the right: 64 channels a workgroup,
// sixteen runs of segments, which join in LDS.
template <bool kGrad>
__global__ void __launch_bounds__(1024) k_join(RecurrenceArgs A) {
    constexpr int kRuns = 16;
    __shared__ float sp[kRuns][64], sy[kRuns][64], sr[kRuns][64];
    const int lane = threadIdx.x % 64, run = threadIdx.x / 64, blocks = (A.channels + 63) / 64;
    const int each = (A.segments + kRuns - 1) / kRuns, first = run * each, last = min(first + each, A.segments);
    for (long long id = blockIdx.x; id < A.batch * blocks; id += gridDim.x) {
        const long long batch = id / blocks;
        const int channel = min(static_cast<int>(id - batch * blocks) * 64 + lane, A.channels - 1);
        const long long state = batch * A.channels + channel, at = batch * A.segments * A.channels + channel;
        float p = 1.f, y = 0.f, r = 0.f;
        for (int s = first; s < last; ++s) {
            const long long i = at + static_cast<long long>(s) * A.channels;
            const float q = A.p[i];
            y = fmaf(q, y, A.y[i]);
            if constexpr (kGrad) r = fmaf(p, A.r[i], r);
            p *= q;
        }
        __syncthreads();
        sp[run][lane] = p, sy[run][lane] = y, sr[run][lane] = r;
        __syncthreads();
        float h = A.initial ? A.initial[state] : 0.f;
        for (int v = 0; v < run; ++v) h = fmaf(sp[v][lane], h, sy[v][lane]);
        for (int s = first; s < last; ++s) {
            const long long i = at + static_cast<long long>(s) * A.channels;
            A.enter[i] = h;
            h = fmaf(A.p[i], h, A.y[i]);
        }
        if constexpr (kGrad) {
            float g = A.grad_end ? A.grad_end[state] : 0.f;
            for (int v = kRuns - 1; v > run; --v) g = fmaf(sp[v][lane], g, sr[v][lane]);
            for (int s = last - 1; s >= first; --s) {
                const long long i = at + static_cast<long long>(s) * A.channels;
                A.leave[i] = g;
                g = fmaf(A.p[i], g, A.r[i]);
            }
            if (run == 0 && A.grad_initial) A.grad_initial[state] = g;
        }
    }
}

// The gradients of kTile steps, from what enters them on both sides.
template <class T, int kC, int kL, bool kJoins>
__global__ void __launch_bounds__(kThreads, kL == 64 ? 4 : 2) k_grad(RecurrenceArgs A) {
    constexpr int kU = hx::kU<kC>, kTile = hx::kTile<kC, kL>, kW = kThreads / kL;
    using Vec = typename Packed<T, kC>::Vec;
    __shared__ float ends[kW][3 * kC][kL];
    const int group = group_of<kL>(), lane = threadIdx.x % kL;
    each_place(A, [&](long long place) {
        const long long id = A.batch * A.segments * A.blocks - 1 - place;     // as above
        const Where w = Where::of<kC, kL>(A, id);
        const int t = w.segment * kTile + group * kU;
        Vec x[kU], g[kU], d[kU];
        fetch<T, kC>(x, A.x, A.x_stride, w, t);
        fetch<T, kC>(g, A.gate, A.gate_stride, w, t);
        fetch<T, kC>(d, A.grad_o, A.grad_o_stride, w, t);
        float h[kC], back[kC];
        w.entering<kJoins>(A, h);
        w.leaving<kJoins>(A, back);
        float z[kU][kC], a[kU][kC], p[kC], y[kC], r[kC];
        // an opening again, from what is held of it
        auto held = [&](auto shuts, int u, int c, bool live) {
            Opening<decltype(shuts)::value> open;
            open.z = z[u][c], open.a = a[u][c];
            open.shut = decltype(shuts)::value && live && part<Vec, kC>(g[u], c) <= kShut;
            return open;
        };
#pragma unroll
        for (int c = 0; c < kC; ++c) p[c] = 1.f, y[c] = r[c] = 0.f;
        auto run = [&](auto whole, auto shuts) {
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const bool live = decltype(whole)::value || t + u < w.length;
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const Opening<decltype(shuts)::value> open(part<Vec, kC>(g[u], c), live);
                    z[u][c] = open.z, a[u][c] = open.a;
                    p[c] = open.left(p[c]);
                    if (live) {                  // what lies past the length may be no number
                        y[c] = open.moved(y[c], part<Vec, kC>(x[u], c));
                        r[c] = fmaf(p[c], part<Vec, kC>(d[u], c), r[c]);
                    }
                }
            }
        };
        const bool whole_group = t + kU <= w.length, some_shut = any_shuts<kC>(g);
        with_kind(whole_group, some_shut, run);
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            ends[group][c][lane] = p[c];
            ends[group][kC + c][lane] = y[c];
            ends[group][2 * kC + c][lane] = r[c];
        }
        __syncthreads();
#pragma unroll 8
        for (int v = 0; v < kW - 1; ++v)
            if (v < group)
#pragma unroll
                for (int c = 0; c < kC; ++c) h[c] = fmaf(ends[v][c][lane], h[c], ends[v][kC + c][lane]);
#pragma unroll 8
        for (int v = kW - 1; v > 0; --v)
            if (v > group)
#pragma unroll
                for (int c = 0; c < kC; ++c) back[c] = fmaf(ends[v][c][lane], back[c], ends[v][2 * kC + c][lane]);
        auto out = [&](auto whole, auto shuts) {
            float off[kU][kC];                   // h_{t-1} - x_t
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const bool live = decltype(whole)::value || t + u < w.length;
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const float v = part<Vec, kC>(x[u], c);
                    off[u][c] = h[c] - v;
                    if (live) h[c] = held(shuts, u, c, live).moved(h[c], v);
                }
            }
            T* dx = static_cast<T*>(A.grad_x) + (w.batch * A.time + t) * A.channels;
            T* dg = static_cast<T*>(A.grad_gate) + (w.batch * A.time + t) * A.channels;
#pragma unroll
            for (int u = kU - 1; u >= 0; --u) {
                const bool live = decltype(whole)::value || t + u < w.length;
                float vx[kC], vg[kC];
#pragma unroll
                for (int c = 0; c < kC; ++c) {
                    const float l = part<Vec, kC>(d[u], c) + back[c], zl = z[u][c] * l;
                    vx[c] = live ? zl : 0.f;
                    vg[c] = live ? a[u][c] * zl * off[u][c] : 0.f;
                    if (live) back[c] = held(shuts, u, c, live).left(l);
                }
                if (decltype(whole)::value || t + u < A.time) {
                    *reinterpret_cast<Vec*>(dx + static_cast<long long>(u) * A.channels + w.channel) = packed<T, kC>(vx);
                    *reinterpret_cast<Vec*>(dg + static_cast<long long>(u) * A.channels + w.channel) = packed<T, kC>(vg);
                }
            }
        };
        with_kind(whole_group, some_shut, out);
        if ((kJoins ? w.segment == 0 : A.segments == 1) && A.grad_initial && group == 0)
#pragma unroll
            for (int c = 0; c < kC; ++c) A.grad_initial[w.batch * A.channels + w.channel + c] = back[c];
    });
}

// One step for a batch of running sequences: kV channels a thread.  64 x 1024 in bf16: 3 us on the
// GPU, 9 for the call.
template <class T, int kV>
__global__ void __launch_bounds__(256) k_step(RecurrenceArgs A, float* states, const int32_t* slots, long long n_slots) {
    const int each = A.channels / kV;
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= A.batch * each) return;
    const long long batch = i / each;
    const int c = static_cast<int>(i - batch * each) * kV;
    const long long slot = slots ? slots[batch] : batch;
    const T* x = static_cast<const T*>(A.x) + batch * A.x_stride[0] + c;
    const T* g = static_cast<const T*>(A.gate) + batch * A.gate_stride[0] + c;
    T* o = static_cast<T*>(A.o) + batch * A.o_stride[0] + c;
    struct alignas(sizeof(T)) Few { T v[kV]; };
    struct alignas(4) Held { float v[kV]; };
    Few out{};
    if (slot >= 0 && slot < n_slots) {
        const Few xs = *reinterpret_cast<const Few*>(x), gs = *reinterpret_cast<const Few*>(g);
        Held* const at = reinterpret_cast<Held*>(states + slot * A.channels + c);
        Held h = *at;
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            h.v[v] = Opening<true>(to_f32(gs.v[v]), true).moved(h.v[v], to_f32(xs.v[v]));
            out.v[v] = from_f32<T>(h.v[v]);
        }
        *at = h;
    } else {
#pragma unroll
        for (int v = 0; v < kV; ++v) out.v[v] = from_f32<T>(0.f);
    }
    *reinterpret_cast<Few*>(o) = out;
}

// How the work is cut: lanes a step's row (kL) and channels a lane (kC), segments of so many steps.
struct Cut { int lanes, channels, segments, steps; };

// Calls f with kC and kL for `channels` channels a lane.
template <class F>
auto with_lanes(int lanes, int channels, F&& f) {
    using One = std::integral_constant<int, 1>;
    if (lanes == 4) return f(One{}, std::integral_constant<int, 4>{});
    if (lanes == 16) return f(One{}, std::integral_constant<int, 16>{});
    if (channels == 1) return f(One{}, std::integral_constant<int, 64>{});
    return f(std::integral_constant<int, 2>{}, std::integral_constant<int, 64>{});
}

// Few channels leave lanes without one: 4 or 16 lanes then take a step's row, and a workgroup's
// groups of them more steps (13 x 9342 x 3 in fp32, with gradient: 50 us, with 64 lanes 76), where
// there are as many steps (2000 x 30 x 4: 156 and 40).
//
// Segments are of whole tiles, the gradient's of one tile each.  Forward, workgroups that walk along
// whole sequences read the data once, those that walk along segments twice; but a walk's tiles come
// one after another, and a CU with one walk waits for its loads.  8 x 4096 x 2048 in bf16: 128
// walks of two channels a lane 123 us, 256 of one 91, 670 MB in segments 137; half of the
// sequences: 76 either way.
Cut cut_of(const hx_recurrence_args& A, bool grad) {
    const int lanes = A.channels <= 4 && A.time >= 1024 ? 4 : A.channels <= 16 && A.time >= 256 ? 16 : 64;
    auto walks = [&](int channels) { return A.batch * ((A.channels + lanes * channels - 1) / (lanes * channels)); };
    const bool wide = A.type != HX_F32 && lanes == 64 && A.channels > 1 && (grad || walks(2) >= 256 || walks(1) < 160);
    const int channels = wide ? 2 : 1;
    const int tile = with_lanes(lanes, channels, [](auto c, auto l) { return kTile<decltype(c)::value, decltype(l)::value>; });
    const long long tiles = std::max<long long>(1, (A.time + tile - 1) / tile);
    long long segments = grad ? tiles : walks(1) >= 160 || tiles <= 4 ? 1 : std::min<long long>(tiles, (512 + walks(channels) - 1) / walks(channels));
    const long long each = (tiles + segments - 1) / segments;
    segments = (tiles + each - 1) / each;
    return {lanes, channels, static_cast<int>(segments), static_cast<int>(each * tile)};
}

// Up to so many segments join those beside them by themselves, which saves a launch (13 x 777 x 601 in
// fp16: 21 us, with it 23; 32 segments of 2 x 2000 x 600: 40 and 38).
constexpr int kJoined = 16;

// The workspace's parts, one after another.
size_t part_bytes(const hx_recurrence_args& A, const Cut& cut) {
    return sizeof(float) * A.batch * cut.segments * A.channels;
}

RecurrenceArgs recurrence_args(const hx_recurrence_args& A, const Cut& cut) {
    RecurrenceArgs R{};
    R.x = A.x, R.gate = A.gate, R.grad_o = A.grad_o;
    R.o = A.o, R.grad_x = A.grad_x, R.grad_gate = A.grad_gate;
    for (int i = 0; i < 2; ++i) {
        R.x_stride[i] = A.x_stride[i], R.gate_stride[i] = A.gate_stride[i];
        R.grad_o_stride[i] = A.grad_o_stride[i], R.o_stride[i] = A.o_stride[i];
    }
    R.lengths = A.lengths, R.initial = A.initial_state, R.grad_end = A.grad_end;
    R.end = A.end_state, R.grad_initial = A.grad_initial;
    R.time = static_cast<int>(A.time), R.channels = static_cast<int>(A.channels), R.batch = A.batch;
    const int width = cut.lanes * cut.channels;
    R.blocks = (R.channels + width - 1) / width;
    R.segments = cut.segments, R.steps = cut.steps;
    // rows that all start at lines of 128 bytes
    const uint64_t size = A.type == HX_F32 ? 4 : 2;
    uint64_t starts = R.channels * size;
    for (const void* p : {R.x, R.gate, R.grad_o, static_cast<const void*>(R.o)}) starts |= reinterpret_cast<uintptr_t>(p);
    for (const long long* s : {R.x_stride, R.gate_stride, R.grad_o_stride, R.o_stride})
        for (int i = 0; i < 2; ++i) starts |= static_cast<uint64_t>(s[i]) * size;
    R.runs = starts % 128 != 0;
    if (cut.segments > 1) {
        float* const space = static_cast<float*>(A.workspace);
        const size_t n = part_bytes(A, cut) / sizeof(float);
        R.p = space, R.y = space + n, R.enter = space + 2 * n, R.r = space + 3 * n, R.leave = space + 4 * n;
    }
    return R;
}

// Calls f(element type, kC, kL).
template <class F>
hipError_t with_cut(const hx_recurrence_args& A, const Cut& cut, F&& f) {
    return with_type(A.type, [&](auto t) {
        return with_lanes(cut.lanes, cut.channels, [&](auto c, auto l) -> hipError_t {
            // two channels a lane are for 16 bits
            if constexpr (std::is_same_v<decltype(t), float> && decltype(c)::value == 2) return hipErrorInvalidValue;
            else return f(t, c, l);
        });
    });
}

// (a multiple of eight, for each_place)
unsigned workgroups(long long n) { return static_cast<unsigned>(std::min<long long>((n + 7) / 8 * 8, 1 << 22)); }

template <bool kGrad>
hipError_t join(const RecurrenceArgs& R, hipStream_t st) {
    k_join<kGrad><<<workgroups(R.batch * ((R.channels + 63) / 64)), 1024, 0, st>>>(R);
    return hipGetLastError();
}

}  // namespace

size_t recurrence_workspace(const hx_recurrence_args& A, bool grad) {
    const Cut cut = cut_of(A, grad);
    return cut.segments > 1 ? (grad ? 5 : 3) * part_bytes(A, cut) : 0;
}

hipError_t recurrence_forward(const hx_recurrence_args& A) {
    const Cut cut = cut_of(A, false);
    const RecurrenceArgs R = recurrence_args(A, cut);
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    const unsigned grid = workgroups(R.batch * R.segments * R.blocks);
    return with_cut(A, cut, [&](auto t, auto c, auto l) -> hipError_t {
        using T = decltype(t);
        constexpr int kC = decltype(c)::value, kL = decltype(l)::value;
        if (R.segments > 1) {
            k_segments<T, kC, kL, false><<<grid, kThreads, 0, st>>>(R);
            hipError_t e = hipGetLastError();
            if (e == hipSuccess && R.segments > kJoined) e = join<false>(R, st);
            if (e != hipSuccess) return e;
        }
        if (R.segments > 1 && R.segments <= kJoined) k_walk<T, kC, kL, true><<<grid, kThreads, 0, st>>>(R);
        else k_walk<T, kC, kL, false><<<grid, kThreads, 0, st>>>(R);
        return hipGetLastError();
    });
}

hipError_t recurrence_backward(const hx_recurrence_args& A) {
    const Cut cut = cut_of(A, true);
    const RecurrenceArgs R = recurrence_args(A, cut);
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    const unsigned grid = workgroups(R.batch * R.segments * R.blocks);
    return with_cut(A, cut, [&](auto t, auto c, auto l) -> hipError_t {
        using T = decltype(t);
        constexpr int kC = decltype(c)::value, kL = decltype(l)::value;
        if (R.segments > 1) {
            k_segments<T, kC, kL, true><<<grid, kThreads, 0, st>>>(R);
            hipError_t e = hipGetLastError();
            if (e == hipSuccess && R.segments > kJoined) e = join<true>(R, st);
            if (e != hipSuccess) return e;
        }
        if (R.segments > 1 && R.segments <= kJoined) k_grad<T, kC, kL, true><<<grid, kThreads, 0, st>>>(R);
        else k_grad<T, kC, kL, false><<<grid, kThreads, 0, st>>>(R);
        return hipGetLastError();
    });
}

hipError_t recurrence_step(const hx_recurrence_args& A) {
    const RecurrenceArgs R = recurrence_args(A, Cut{64, 1, 1, 1});
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    const int v = A.channels % 4 == 0 ? 4 : 1;
    const unsigned grid = static_cast<unsigned>((A.batch * (A.channels / v) + 255) / 256);
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        if (v == 4) k_step<T, 4><<<grid, 256, 0, st>>>(R, A.state, A.slots, A.n_slots);
        else k_step<T, 1><<<grid, 256, 0, st>>>(R, A.state, A.slots, A.n_slots);
        return hipGetLastError();
    });
}

}  // namespace hx
