// Layer norm of rows, and its gradient.
//
// A row is read once, held in registers, and written once: kGroup lanes hold it in kV pieces of
// 16 bytes each.  The variance is the mean square of differences from a first mean, which their own
// sum then corrects (sums over the held row, not the difference of two large numbers).  Workgroups walk over the rows, so that
// weight and bias stay in registers too, and the gradients of both are added there: each
// workgroup writes its sums once, a second launch adds those up in a fixed order.  (Few rows are
// read a second time instead, by columns.)  Both are bound by the rows' bytes: 32768 x 4096 in
// bf16 forward 96 us, 5.6 TB/s, backward 156, 5.2, and 5 for the sums (a copy: 4.9).
#include "readout.h"

#include <algorithm>
#include <type_traits>

namespace hx {
namespace {

struct NormArgs {
    const void *x, *dy;
    void* y;                         // or dx
    long long x_stride, dy_stride, y_stride;
    const void *weight, *bias;
    int weight_type, width;
    long long rows;
    float eps, per_width;
    float *mean, *rstd;
    float* part;                     // (workgroups, 2, width): sums of dy n, of dy
};

// kE elements of a row from element j on, wherever they start, as fp32.
template <class T, int kE> struct Piece { typedef typename PieceOf<T>::Vec Vec; };
template <> struct Piece<float, 8> { typedef float Vec __attribute__((ext_vector_type(8), aligned(4))); };
template <class T> struct Piece<T, 1> { typedef T Vec; };
template <> struct Piece<__half, 2> { typedef _Float16 Vec __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Piece<__hip_bfloat16, 2> { typedef __bf16 Vec __attribute__((ext_vector_type(2), aligned(2))); };
template <> struct Piece<__half, 4> { typedef _Float16 Vec __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Piece<__hip_bfloat16, 4> { typedef __bf16 Vec __attribute__((ext_vector_type(4), aligned(2))); };

template <class T, int kE>
__device__ __forceinline__ void widen(const typename Piece<T, kE>::Vec& raw, float* v) {
    if constexpr (kE == 1) {
        v[0] = to_f32(raw);
    } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) v[i] = static_cast<float>(raw[i]);
    }
}

template <class T, int kE>
__device__ __forceinline__ void store(T* to, const float* v) {
    typename Piece<T, kE>::Vec raw;
    if constexpr (kE == 1) {
        raw = from_f32<T>(v[0]);
    } else {
#pragma unroll
        for (int i = 0; i < kE; ++i) raw[i] = static_cast<decltype(raw[0] + raw[0])>(v[i]);
    }
    *reinterpret_cast<typename Piece<T, kE>::Vec*>(to) = raw;
}

template <int kE>
__device__ __forceinline__ void load_weights(const void* w, int type, int j, float* v) {
    auto as = [&](auto t) {
        using W = decltype(t);
        widen<W, kE>(*reinterpret_cast<const typename Piece<W, kE>::Vec*>(static_cast<const W*>(w) + j), v);
    };
    if (type == HX_F16) as(__half{});
    else if (type == HX_BF16) as(__hip_bfloat16{});
    else as(float{});
}

// Sums of kN values over the kGroup lanes (of kThreads) that share a row; every lane gets them.
// Between two calls with the same sh lies a call with another, so that one barrier is enough.
template <int kGroup, int kN>
__device__ __forceinline__ void group_sum(float (&x)[kN], float* sh) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
        for (int m = (kGroup < 64 ? kGroup : 64) / 2; m > 0; m >>= 1) x[n] += __shfl_xor(x[n], m);
    if constexpr (kGroup > 64) {
        constexpr int kWaves = kGroup / 64;
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int n = 0; n < kN; ++n) sh[n * kWaves + threadIdx.x / 64] = x[n];
        __syncthreads();
#pragma unroll
        for (int n = 0; n < kN; ++n) {
            x[n] = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) x[n] += sh[n * kWaves + w];
        }
    }
}

// Where a lane's piece k starts, and how many of its first elements belong to the piece before it:
// the last piece of a row that is no whole number of pieces is its last kE elements.
template <int kE, int kGroup, bool kRagged>
struct Place {
    int at, skip;
    bool here;
    __device__ __forceinline__ Place(int width, int lane, int k) {
        const int p = lane + k * kGroup, whole = width / kE;
        here = p < whole;
        at = p * kE, skip = 0;
        if constexpr (kRagged) {
            if (p == whole) here = true, at = width - kE, skip = kE - width % kE;
        }
    }
};

// From the sums of the differences from a first mean, and of their squares: what that mean was off by
// (a sum of 500 voltages near -65 is off by their own 2^-24 many times over, their differences' is not)
// and 1 / sqrt(variance + eps).
struct Spread {
    float rest, rstd;
    __device__ __forceinline__ Spread(const float (&off)[2], const NormArgs& A) {
        rest = off[0] * A.per_width;
        const float variance = off[1] * A.per_width - rest * rest;
        rstd = 1.f / sqrtf((variance < 0.f ? 0.f : variance) + A.eps);
    }
};

template <class T, int kE, int kGroup, int kV, bool kRagged>
__global__ void __launch_bounds__(kGroup < 256 ? 256 : kGroup) k_norm(NormArgs A) {
    constexpr int kThreads = kGroup < 256 ? 256 : kGroup, kRows = kThreads / kGroup;
    using Vec = typename Piece<T, kE>::Vec;
    using At = Place<kE, kGroup, kRagged>;
    __shared__ float sh[2][2 * 16];
    const int lane = threadIdx.x % kGroup;
    float w[kV][kE], b[kV][kE];
#pragma unroll
    for (int k = 0; k < kV; ++k) {
        const At at(A.width, lane, k);
#pragma unroll
        for (int i = 0; i < kE; ++i) w[k][i] = 1.f, b[k][i] = 0.f;
        if (at.here && A.weight) load_weights<kE>(A.weight, A.weight_type, at.at, w[k]);
        if (at.here && A.bias) load_weights<kE>(A.bias, A.weight_type, at.at, b[k]);
    }
    const long long step = static_cast<long long>(gridDim.x) * kRows;
    long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / kGroup;
    Vec next[kV];
    auto fetch = [&](long long r) {
        const T* x = static_cast<const T*>(A.x) + r * A.x_stride;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
            if (at.here) next[k] = *reinterpret_cast<const Vec*>(x + at.at);
        }
    };
    if (row < A.rows) fetch(row);
    for (; row < A.rows; row += step) {
        float v[kV][kE], sum[1] = {0.f}, off[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
            widen<T, kE>(next[k], v[k]);
#pragma unroll
            for (int i = 0; i < kE; ++i) sum[0] += at.here && i >= at.skip ? v[k][i] : 0.f;
        }
        if (row + step < A.rows) fetch(row + step);
        group_sum<kGroup>(sum, sh[0]);
        const float mean = sum[0] * A.per_width;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                v[k][i] -= mean;
                off[0] += at.here && i >= at.skip ? v[k][i] : 0.f;
                off[1] += at.here && i >= at.skip ? v[k][i] * v[k][i] : 0.f;
            }
        }
        group_sum<kGroup>(off, sh[1]);
        const Spread spread(off, A);
        const float rest = spread.rest, rstd = spread.rstd;
        if (lane == 0) {
            A.mean[row] = mean + rest;
            A.rstd[row] = rstd;
        }
        T* y = static_cast<T*>(A.y) + row * A.y_stride;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
#pragma unroll
            for (int i = 0; i < kE; ++i) v[k][i] = fmaf((v[k][i] - rest) * rstd, w[k][i], b[k][i]);
            if (at.here) store<T, kE>(y + at.at, v[k]);
        }
    }
}

template <class T, int kE, int kGroup, int kV, bool kRagged, bool kSums>
__global__ void __launch_bounds__(kGroup < 256 ? 256 : kGroup) k_norm_grad(NormArgs A) {
    constexpr int kThreads = kGroup < 256 ? 256 : kGroup, kRows = kThreads / kGroup;
    using Vec = typename Piece<T, kE>::Vec;
    using At = Place<kE, kGroup, kRagged>;
    __shared__ float sh[2][2 * 16];
    const int lane = threadIdx.x % kGroup;
    float w[kV][kE], dw[kV][kE], db[kV][kE];
#pragma unroll
    for (int k = 0; k < kV; ++k) {
        const At at(A.width, lane, k);
#pragma unroll
        for (int i = 0; i < kE; ++i) w[k][i] = 1.f, dw[k][i] = db[k][i] = 0.f;
        if (at.here && A.weight) load_weights<kE>(A.weight, A.weight_type, at.at, w[k]);
    }
    const long long step = static_cast<long long>(gridDim.x) * kRows;
    long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / kGroup;
    Vec next_x[kV], next_dy[kV];
    float next_mean = 0.f, next_rstd = 0.f;
    auto fetch = [&](long long r) {
        const T* x = static_cast<const T*>(A.x) + r * A.x_stride;
        const T* dy = static_cast<const T*>(A.dy) + r * A.dy_stride;
        next_mean = A.mean[r], next_rstd = A.rstd[r];
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
            if (at.here) {
                next_x[k] = *reinterpret_cast<const Vec*>(x + at.at);
                next_dy[k] = *reinterpret_cast<const Vec*>(dy + at.at);
            }
        }
    };
    if (row < A.rows) fetch(row);
    for (int turn = 0; row < A.rows; row += step, turn ^= 1) {
        const float mean = next_mean, rstd = next_rstd;
        float n[kV][kE], g[kV][kE], sum[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
            float v[kE], d[kE];
            widen<T, kE>(next_x[k], v);
            widen<T, kE>(next_dy[k], d);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                n[k][i] = (v[i] - mean) * rstd;
                g[k][i] = d[i] * w[k][i];
                if (at.here && i >= at.skip) {
                    sum[0] += g[k][i];
                    sum[1] = fmaf(g[k][i], n[k][i], sum[1]);
                    if constexpr (kSums) {
                        dw[k][i] = fmaf(d[i], n[k][i], dw[k][i]);
                        db[k][i] += d[i];
                    }
                }
            }
        }
        if (row + step < A.rows) fetch(row + step);
        group_sum<kGroup>(sum, sh[turn]);
        const float mean_g = sum[0] * A.per_width, mean_gn = sum[1] * A.per_width;
        T* dx = static_cast<T*>(A.y) + row * A.y_stride;
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
            float v[kE];
#pragma unroll
            for (int i = 0; i < kE; ++i) v[i] = rstd * (g[k][i] - mean_g - n[k][i] * mean_gn);
            if (at.here) store<T, kE>(dx + at.at, v);
        }
    }
    if constexpr (!kSums) return;
    float* part = A.part + static_cast<long long>(blockIdx.x) * 2 * A.width;
    if constexpr (kRows == 1) {
#pragma unroll
        for (int k = 0; k < kV; ++k) {
            const At at(A.width, lane, k);
            if (at.here)
#pragma unroll
                for (int i = 0; i < kE; ++i)
                    if (i >= at.skip) {
                        part[at.at + i] = dw[k][i];
                        part[A.width + at.at + i] = db[k][i];
                    }
        }
    } else {
        // the workgroup's groups of lanes hold the same columns: added in LDS, column by column
        constexpr int kHeld = kGroup * kV * kE;
        __shared__ float held[kRows * kHeld];
        const int group = threadIdx.x / kGroup;
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                const At at(A.width, lane, k);
                if (at.here)
#pragma unroll
                    for (int i = 0; i < kE; ++i)
                        if (i >= at.skip) held[group * kHeld + at.at + i] = which ? db[k][i] : dw[k][i];
            }
            __syncthreads();
            for (int j = threadIdx.x; j < A.width; j += kThreads) {
                float s = 0.f;
                for (int r = 0; r < kRows; ++r) s += held[r * kHeld + j];
                part[which * A.width + j] = s;
            }
        }
    }
}

// Rows too wide for registers: read again from the cache for each sum.  A thread adds a piece's terms in
// fp32 and pieces, of which there may be thousands, in 64 bits.
constexpr int kWide = 1024;

template <class T, class F>
__device__ __forceinline__ void each_element(int width, F f) {
    constexpr int kE = sizeof(typename PieceOf<T>::Vec) / sizeof(T);
    for (int j = threadIdx.x * kE; j + kE <= width; j += kWide * kE) f(std::integral_constant<int, kE>{}, j);
    const int j = width / kE * kE + threadIdx.x;
    if (j < width) f(std::integral_constant<int, 1>{}, j);
}

template <class T, int kE>
__device__ __forceinline__ void load(const T* from, float* v) {
    widen<T, kE>(*reinterpret_cast<const typename Piece<T, kE>::Vec*>(from), v);
}

template <class T>
__global__ void __launch_bounds__(kWide) k_norm_wide(NormArgs A) {
    __shared__ float sh[2][2 * 16];
    for (long long row = blockIdx.x; row < A.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(A.x) + row * A.x_stride;
        T* y = static_cast<T*>(A.y) + row * A.y_stride;
        double own = 0., own_off[2] = {0., 0.};
        each_element<T>(A.width, [&](auto e, int j) {
            constexpr int kE = decltype(e)::value;
            float v[kE], s = 0.f;
            load<T, kE>(x + j, v);
#pragma unroll
            for (int i = 0; i < kE; ++i) s += v[i];
            own += s;
        });
        float sum[1] = {static_cast<float>(own)};
        group_sum<kWide>(sum, sh[0]);
        const float mean = sum[0] * A.per_width;
        each_element<T>(A.width, [&](auto e, int j) {
            constexpr int kE = decltype(e)::value;
            float v[kE], s = 0.f, d = 0.f;
            load<T, kE>(x + j, v);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                d += v[i] - mean;
                s = fmaf(v[i] - mean, v[i] - mean, s);
            }
            own_off[0] += d;
            own_off[1] += s;
        });
        float off[2] = {static_cast<float>(own_off[0]), static_cast<float>(own_off[1])};
        group_sum<kWide>(off, sh[1]);
        const Spread spread(off, A);
        const float rest = spread.rest, rstd = spread.rstd;
        if (threadIdx.x == 0) {
            A.mean[row] = mean + rest;
            A.rstd[row] = rstd;
        }
        each_element<T>(A.width, [&](auto e, int j) {
            constexpr int kE = decltype(e)::value;
            float v[kE], w[kE], b[kE];
            load<T, kE>(x + j, v);
#pragma unroll
            for (int i = 0; i < kE; ++i) w[i] = 1.f, b[i] = 0.f;
            if (A.weight) load_weights<kE>(A.weight, A.weight_type, j, w);
            if (A.bias) load_weights<kE>(A.bias, A.weight_type, j, b);
#pragma unroll
            for (int i = 0; i < kE; ++i) v[i] = fmaf((v[i] - mean - rest) * rstd, w[i], b[i]);
            store<T, kE>(y + j, v);
        });
    }
}

template <class T>
__global__ void __launch_bounds__(kWide) k_norm_grad_wide(NormArgs A) {
    __shared__ float sh[2][2 * 16];
    int turn = 0;
    for (long long row = blockIdx.x; row < A.rows; row += gridDim.x, turn ^= 1) {
        const T* x = static_cast<const T*>(A.x) + row * A.x_stride;
        const T* dy = static_cast<const T*>(A.dy) + row * A.dy_stride;
        T* dx = static_cast<T*>(A.y) + row * A.y_stride;
        const float mean = A.mean[row], rstd = A.rstd[row];
        double own[2] = {0., 0.};
        auto terms = [&](auto e, int j, float* n, float* g) {
            constexpr int kE = decltype(e)::value;
            float w[kE];
            load<T, kE>(x + j, n);
            load<T, kE>(dy + j, g);
#pragma unroll
            for (int i = 0; i < kE; ++i) w[i] = 1.f;
            if (A.weight) load_weights<kE>(A.weight, A.weight_type, j, w);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                n[i] = (n[i] - mean) * rstd;
                g[i] *= w[i];
            }
        };
        each_element<T>(A.width, [&](auto e, int j) {
            constexpr int kE = decltype(e)::value;
            float n[kE], g[kE], s = 0.f, sn = 0.f;
            terms(e, j, n, g);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                s += g[i];
                sn = fmaf(g[i], n[i], sn);
            }
            own[0] += s;
            own[1] += sn;
        });
        float sum[2] = {static_cast<float>(own[0]), static_cast<float>(own[1])};
        group_sum<kWide>(sum, sh[turn]);
        const float mean_g = sum[0] * A.per_width, mean_gn = sum[1] * A.per_width;
        each_element<T>(A.width, [&](auto e, int j) {
            constexpr int kE = decltype(e)::value;
            float n[kE], g[kE];
            terms(e, j, n, g);
#pragma unroll
            for (int i = 0; i < kE; ++i) n[i] = rstd * (g[i] - mean_g - n[i] * mean_gn);
            store<T, kE>(dx + j, n);
        });
    }
}

// Rows whose terms of a column's sum are added one after another in fp32: gradients that are alike have
// roundings that are, too.  What follows is added in 64 bits.
constexpr int kChain = 128;

// Sums of dy n and of dy over a run of rows, kE columns a thread.
template <class T, int kE>
__global__ void __launch_bounds__(256) k_norm_columns(NormArgs A, long long rows_each, float* dw, float* db) {
    // threads past the last column do the last columns over again
    const int j = min((static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x)) * kE, A.width - kE);
    const long long first = blockIdx.y * rows_each, end = min(first + rows_each, A.rows);
    const T* x = static_cast<const T*>(A.x) + j;
    const T* dy = static_cast<const T*>(A.dy) + j;
    double whole[2][kE] = {};
    for (long long r0 = first; r0 < end; r0 += kChain) {
        const long long last = min(r0 + kChain, end);
        float sum[2][kE] = {};
#pragma unroll 8
        for (long long r = r0; r < last; ++r) {
            float v[kE], d[kE];
            load<T, kE>(x + r * A.x_stride, v);
            load<T, kE>(dy + r * A.dy_stride, d);
            const float mean = A.mean[r], rstd = A.rstd[r];
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                sum[0][i] = fmaf(d[i], (v[i] - mean) * rstd, sum[0][i]);
                sum[1][i] += d[i];
            }
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) whole[0][i] += sum[0][i], whole[1][i] += sum[1][i];
    }
    dw += static_cast<long long>(blockIdx.y) * 2 * A.width + j;
    db += static_cast<long long>(blockIdx.y) * 2 * A.width + j;
#pragma unroll
    for (int i = 0; i < kE; ++i) dw[i] = static_cast<float>(whole[0][i]), db[i] = static_cast<float>(whole[1][i]);
}

// The workgroups' sums, added up: 32 columns a workgroup, 32 runs of rows each.
__global__ void __launch_bounds__(1024) k_norm_join(const float* part, int parts, int width, float* dw, float* db) {
    constexpr int kColumns = 32, kRuns = 32;
    __shared__ double sh[kRuns][kColumns + 1];
    const long long whole = 2LL * width, column = static_cast<long long>(blockIdx.x) * kColumns + threadIdx.x % kColumns;
    const int run = threadIdx.x / kColumns;
    double s = 0.;
    if (column < whole) {
#pragma unroll 8
        for (int p = run; p < parts; p += kRuns) s += part[p * whole + column];
    }
    sh[run][threadIdx.x % kColumns] = s;
    __syncthreads();
    // the 32 runs of a column lie across half a wave
    s = sh[threadIdx.x % kRuns][threadIdx.x / kRuns];
    for (int d = kRuns / 2; d > 0; d >>= 1) s += __shfl_xor(s, d);
    const long long mine = static_cast<long long>(blockIdx.x) * kColumns + threadIdx.x / kRuns;
    if (threadIdx.x % kRuns == 0 && mine < whole) (mine < width ? dw[mine] : db[mine - width]) = static_cast<float>(s);
}

// How a row is held: kE elements a piece, kGroup lanes, kV pieces a lane.
template <int E, int G, int V>
struct Shape {
    static constexpr int kE = E, kGroup = G, kV = V, kThreads = G < 256 ? 256 : G, kRows = kThreads / (G ? G : 256);
};
using TooWide = Shape<0, 0, 0>;

// Calls f with the Shape for rows of this width.
template <class T, bool kGrad, class F>
auto with_shape(int width, F&& f) {
    constexpr int kE = sizeof(typename PieceOf<T>::Vec) / sizeof(T);
    const int pieces = (width + kE - 1) / kE;
    if (width < kE) return f(Shape<1, 8, 1>{});
    if (pieces <= 8) return f(Shape<kE, 8, 1>{});
    if (pieces <= 16) return f(Shape<kE, 8, 2>{});
    if (pieces <= 64) return f(Shape<kE, 64, 1>{});
    if (pieces <= 128) return f(Shape<kE, 64, 2>{});
    if (pieces <= 256) return f(Shape<kE, 256, 1>{});
    if (pieces <= 512) return f(Shape<kE, 256, 2>{});
    // The gradient holds two rows and two sums: 16 elements a lane of 1024 lanes are more than the
    // registers hold, 12 are not (4032 x 8587 in fp16, with the forward pass: 222 us and 128).
    if constexpr (kGrad) {
        if (pieces <= 1024) return f(std::conditional_t<kE == 8, Shape<8, 1024, 1>, Shape<4, 256, 4>>{});
        if (width <= 8 * 1024) return f(Shape<4, 1024, 2>{});
        if (width <= 12 * 1024) return f(Shape<4, 1024, 3>{});
    } else {
        if (pieces <= 1024) return f(Shape<kE, 256, 4>{});
        if (pieces <= 2048) return f(Shape<kE, 1024, 2>{});
        if constexpr (kE == 4)
            if (pieces <= 4096) return f(Shape<4, 1024, 4>{});
    }
    return f(TooWide{});
}

NormArgs norm_args(const hx_norm_args& A) {
    NormArgs N{};
    N.x = A.x, N.x_stride = A.x_stride;
    N.weight = A.weight, N.bias = A.bias, N.weight_type = static_cast<int>(A.weight_type);
    N.width = static_cast<int>(A.width), N.rows = A.rows;
    N.eps = static_cast<float>(A.eps), N.per_width = static_cast<float>(1.0 / static_cast<double>(A.width));
    N.mean = A.mean, N.rstd = A.rstd;
    return N;
}

// How the gradients of weight and bias are summed: `held` by the workgroups that make grad_x, one
// sum of each for each of `parts`, of kChain turns at most; or by a launch over the columns that reads the rows again, in
// `parts` runs of rows.
//
// A workgroup's sums are 8 bytes a column, written and read again: more than the rows, where there
// are few.  462 x 11764 in fp16: 75 us held, 31 by columns; 5003 x 1001: 22 held.
struct Sums { bool held; int parts; };

Sums sums_of(const hx_norm_args& A) {
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        return with_shape<T, true>(static_cast<int>(A.width), [&](auto shape) -> Sums {
            using S = decltype(shape);
            if constexpr (S::kE != 0) {
                const int64_t turns = (A.rows + S::kRows - 1) / S::kRows;
                const int64_t parts = std::min<int64_t>({turns, std::max<int64_t>(512, (turns + kChain - 1) / kChain), 1 << 21});
                if (A.rows * static_cast<int64_t>(sizeof(T)) >= 8 * parts) return {true, static_cast<int>(parts)};
            }
            const int64_t blocks = (A.width + 511) / 512;
            const int64_t most = std::max<int64_t>(1, 512 / blocks);
            return {false, static_cast<int>(std::max<int64_t>(1, std::min({(A.rows + 15) / 16, most, int64_t(64)})))};
        });
    });
}

}  // namespace

size_t norm_workspace(const hx_norm_args& A) {
    if (!A.grad_weight) return 0;
    const Sums sums = sums_of(A);
    // a single run of rows writes to the gradients themselves
    return sums.held || sums.parts > 1 ? sizeof(float) * 2 * sums.parts * static_cast<size_t>(A.width) : 0;
}

hipError_t norm_forward(const hx_norm_args& A) {
    NormArgs N = norm_args(A);
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    N.y = A.y, N.y_stride = A.y_stride;
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        return with_shape<T, false>(N.width, [&](auto shape) {
            using S = decltype(shape);
            if constexpr (!S::kE) {
                k_norm_wide<T><<<static_cast<unsigned>(std::min<long long>(N.rows, 1 << 16)), kWide, 0, st>>>(N);
            } else {
                const long long turns = (N.rows + S::kRows - 1) / S::kRows;
                const unsigned grid = static_cast<unsigned>(std::min<long long>(turns, 256 * 2048 / S::kThreads));
                if (N.width % S::kE) k_norm<T, S::kE, S::kGroup, S::kV, true><<<grid, S::kThreads, 0, st>>>(N);
                else k_norm<T, S::kE, S::kGroup, S::kV, false><<<grid, S::kThreads, 0, st>>>(N);
            }
            return hipGetLastError();
        });
    });
}

hipError_t norm_backward(const hx_norm_args& A) {
    NormArgs N = norm_args(A);
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    N.dy = A.grad_y, N.dy_stride = A.grad_y_stride, N.y = A.grad_x, N.y_stride = A.grad_x_stride;
    const Sums sums = sums_of(A);
    const bool joined = A.grad_weight && (sums.held || sums.parts > 1);
    float* const part = static_cast<float*>(A.workspace);
    if (A.grad_weight && sums.held) N.part = part;
    hipError_t e = !A.rows ? hipSuccess : with_type(A.type, [&](auto t) {
        using T = decltype(t);
        return with_shape<T, true>(N.width, [&](auto shape) {
            using S = decltype(shape);
            if constexpr (!S::kE) {
                k_norm_grad_wide<T><<<static_cast<unsigned>(std::min<long long>(N.rows, 1 << 16)), kWide, 0, st>>>(N);
            } else {
                const long long turns = (N.rows + S::kRows - 1) / S::kRows;
                const unsigned grid = static_cast<unsigned>(N.part ? sums.parts : std::min<long long>(turns, 256 * 1024 / S::kThreads));
                auto go = [&](auto ragged, auto with_sums) {
                    k_norm_grad<T, S::kE, S::kGroup, S::kV, decltype(ragged)::value, decltype(with_sums)::value>
                        <<<grid, S::kThreads, 0, st>>>(N);
                };
                const bool ragged = N.width % S::kE;
                if (N.part) ragged ? go(std::true_type{}, std::true_type{}) : go(std::false_type{}, std::true_type{});
                else ragged ? go(std::true_type{}, std::false_type{}) : go(std::false_type{}, std::false_type{});
            }
            return hipGetLastError();
        });
    });
    if (e != hipSuccess || !A.grad_weight) return e;
    if (!sums.held && A.rows) {
        float* const dw = joined ? part : A.grad_weight;
        float* const db = joined ? part + A.width : A.grad_bias;
        e = with_type(A.type, [&](auto t) {
            using T = decltype(t);
            const long long each = (A.rows + sums.parts - 1) / sums.parts;
            auto go = [&](auto columns) {
                constexpr int kE = decltype(columns)::value;
                const dim3 grid((N.width + 256 * kE - 1) / (256 * kE), sums.parts);
                k_norm_columns<T, kE><<<grid, 256, 0, st>>>(N, each, dw, db);
            };
            if constexpr (sizeof(T) == 2)
                if (N.width > 1) {
                    go(std::integral_constant<int, 2>{});
                    return hipGetLastError();
                }
            go(std::integral_constant<int, 1>{});
            return hipGetLastError();
        });
        if (e != hipSuccess) return e;
    }
    // without rows the sums are 0
    if (joined || !A.rows)
        k_norm_join<<<static_cast<unsigned>((2 * A.width + 31) / 32), 1024, 0, st>>>(part, A.rows ? sums.parts : 0, N.width,
                                                                                   A.grad_weight, A.grad_bias);
    return hipGetLastError();
}

}  // namespace hx
