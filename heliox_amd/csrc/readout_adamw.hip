// One AdamW step over many tensors.
//
// A workgroup takes kChunk elements of one tensor, a wave kBlocks blocks of 256 in a row, four
// elements a lane in each, so that every array streams through as it lies in memory: bound by
// their bytes (300 tensors of 150 million bf16 elements, 8 bits: 315 us, 4.8 TB/s, 332 where codes are
// rounded by chance; with four blocks a wave 327, with one 333).  The tensors of a launch are listed in
// its arguments; a workgroup finds its own by one comparison a lane.  The count of steps, and what
// follows from it alone, is made by a first launch of one thread, on the device, so that a captured
// step counts on.
//
// In 8 bits a block's moments are e4m3 numbers relative to the block's largest (a wave holds a
// block: its maximum is a reduction of the wave).  Of v the root is held: half of v's exponents, so that
// its 3 bits of mantissa are off by 2^-4 in the step and not in its square.  A root that would
// round to zero is held as the least number instead: a step that divides by too little has no bound.
//
// A moment that moves by less than half a step of its code would never move if it were rounded to
// nearest: with beta2 = 0.999 a root falls by 0.05% a step, and codes are 6 to 12% apart (5000 steps
// after 16384 gradients' sizes changed places a third of the roots were off by more than 2).  So
// a code is rounded up as often as its number is near the upper one, by bits made of the
// step's count and the element's place: the moments follow on average (of those roots 0.3% are off by more
// than 2), and the same calls give the same state.  The first steps, as many as the longer memory
// spans, 1 / (1 - beta), are to nearest: moments of few gradients move by whole codes, and what sticks all
// the same is forgotten in as many steps more.
#include "readout.h"

#include <algorithm>
#include <cmath>

namespace hx {
namespace {

constexpr int kThreads = 256, kBlocks = 2, kBlock = 256, kChunk = kThreads / 64 * kBlocks * kBlock;
constexpr int kTensors = 64;                       // of a launch: a lane each, 3 KB of arguments
constexpr float kTop8 = 448.f, kLeast8 = 0x1p-9f;  // of e4m3
constexpr float kTiny = 0x1p-100f;                 // blocks whose largest moment is below are zero

struct Tensor {
    void* param;
    const void* grad;
    long long elements, start;
    unsigned first;                                // workgroup of the launch
    float decay;
};

// What a step's count and its rates come to, made by k_count.
struct Rates { float size, root; };                // lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t)

struct AdamwArgs {
    Tensor tensor[kTensors];
    int count;
    void *m, *v;
    float *m_scale, *v_scale;
    float beta1, beta2, less1, less2, eps, lr, grad_scale;     // less: 1 - beta
    const int64_t* step;
    int64_t nearest;                                           // steps that round codes to nearest
    const float *grad_scale_ptr, *lr_ptr;
    const Rates* rates;
};

__global__ void k_count(int64_t* step, double log1, double log2, float lr, const float* lr_ptr) {
    const int64_t t = step[0] + 1;
    step[0] = t;
    if (lr_ptr) lr = *lr_ptr;
    Rates r;
    r.size = static_cast<float>(lr / -expm1(t * log1));
    r.root = static_cast<float>(1. / sqrt(-expm1(t * log2)));
    *reinterpret_cast<Rates*>(step + 1) = r;
}

// Four elements, wherever they start.
template <class T> struct Four;
template <> struct Four<float> { typedef float Vec __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Four<__half> { typedef _Float16 Vec __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Four<__hip_bfloat16> { typedef __bf16 Vec __attribute__((ext_vector_type(4), aligned(2))); };
typedef float Float4 __attribute__((ext_vector_type(4)));

template <class T, bool kWhole>
__device__ __forceinline__ Float4 load(const T* at, long long left) {
    Float4 x = {};
    if (kWhole || left >= 4) {
        const auto raw = *reinterpret_cast<const typename Four<T>::Vec*>(at);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(raw[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) x[i] = to_f32(at[i]);
    }
    return x;
}

template <class T, bool kWhole>
__device__ __forceinline__ void store(T* at, Float4 x, long long left) {
    if (kWhole || left >= 4) {
        typename Four<T>::Vec raw;
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = static_cast<decltype(raw[0] + raw[0])>(x[i]);
        *reinterpret_cast<typename Four<T>::Vec*>(at) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) at[i] = from_f32<T>(x[i]);
    }
}

// The largest of a wave's values, none of them negative.
__device__ __forceinline__ float wave_max(float x) {
    auto step = [&](auto control) {
        const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(control)::value, 0xf, 0xf, true);
        x = fmaxf(x, __int_as_float(y));
    };
    step(std::integral_constant<int, 0x111>{});    // rows of 16 lanes: from 1, 2, 4 and 8 lanes to the left
    step(std::integral_constant<int, 0x112>{});
    step(std::integral_constant<int, 0x114>{});
    step(std::integral_constant<int, 0x118>{});
    step(std::integral_constant<int, 0x142>{});    // a row's last lane to the next row, the second's to the last two
    step(std::integral_constant<int, 0x143>{});
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

__device__ __forceinline__ Float4 unpack(int code, float scale) {
    typedef float Two __attribute__((ext_vector_type(2)));
    const Two a = __builtin_amdgcn_cvt_pk_f32_fp8(code, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(code, true);
    return Float4{a.x * scale, a.y * scale, b.x * scale, b.y * scale};
}

__device__ __forceinline__ int pack(Float4 x) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], low, true);
}

// 32 bits for each four elements of a step: a sum of place and count times odd numbers (the first bits
// of the fractions of the square roots of 2, 3, 11 and 17), mixed by shifts and products.  The four turn
// them by 8 bits each and take the upper 16 for the root, the lower for m: what they share
// does not bias either.
constexpr unsigned kRoot2 = 0x6a09e667u, kRoot3 = 0xbb67ae85u, kRoot11 = 0x510e527fu, kRoot17 = 0x1f83d9abu;
__device__ __forceinline__ unsigned mixed(unsigned h) {
    h = (h ^ h >> 16) * kRoot11;
    h = (h ^ h >> 15) * kRoot17;
    return h ^ h >> 16;
}

// Each rounded up where the 20 bits that its code drops and 20 of chance, of which 16 are the element's
// own, add up to 2^20.  16 tell changes of 2^-16 of a code's step, as roots' with beta2 up to 0.9999.
template <bool kHigh>
__device__ __forceinline__ int pack(Float4 x, unsigned bits) {
    auto chance = [&](int i) {
        const unsigned one = __builtin_rotateleft32(bits, 8 * i);
        return (kHigh ? one & 0xffff0000u : one << 16) | 0x8000u;
    };
    int code = __builtin_amdgcn_cvt_sr_fp8_f32(x[0], chance(0), 0, 0);
    code = __builtin_amdgcn_cvt_sr_fp8_f32(x[1], chance(1), code, 1);
    code = __builtin_amdgcn_cvt_sr_fp8_f32(x[2], chance(2), code, 2);
    return __builtin_amdgcn_cvt_sr_fp8_f32(x[3], chance(3), code, 3);
}

// Codes of a block, relative to its largest; that over 448 is returned.  `bits`: of these four elements, where
// codes are not rounded to nearest.
//
// A number next to the middle of two codes goes to one or the other by its last bit, and a block's
// largest number that does so moves the scale of all by a sixteenth.  So that a state's way can be
// followed by any other fp32 arithmetic, moments and quotients are rounded operation by operation, and
// the quotient x / top is the correctly rounded one: from the correctly rounded 1 / top, corrected by
// the exact remainder (Markstein's division).
template <bool kRoot>
__device__ __forceinline__ float quantise(Float4 x, int& code, bool dither, unsigned bits) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(x[i]));
    top = wave_max(top);
    const bool live = top >= kTiny;
    const float per = live ? 1.f / top : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float q = x[i] * per;
        q = fmaf(fmaf(-q, top, x[i]), per, q);
        x[i] = q * kTop8;
        if (kRoot && x[i] > 0.f && x[i] < kLeast8) x[i] = kLeast8;
    }
    code = dither ? pack<kRoot>(x, bits) : pack(x);
    return live ? top * (1.f / kTop8) : 0.f;
}

template <class P, class G, int kBits>
__global__ void __launch_bounds__(kThreads) k_adamw(AdamwArgs A) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    // the last tensor whose first workgroup is not after this one (read through the arguments'
    // pointer: indexed as a value they would be copied to scratch)
    const auto* all = reinterpret_cast<const AdamwArgs*>((const void*)__builtin_amdgcn_kernarg_segment_ptr());
    const bool mine = lane < A.count && all->tensor[lane < A.count ? lane : 0].first <= blockIdx.x;
    const int which = __popcll(__ballot(mine)) - 1;
    const Tensor& t = all->tensor[which];
    const long long base = static_cast<long long>(blockIdx.x - t.first) * kChunk + wave * (kBlocks * kBlock);
    const float lr = A.lr_ptr ? *A.lr_ptr : A.lr, clip = A.grad_scale_ptr ? *A.grad_scale_ptr : A.grad_scale;
    const Rates rates = *A.rates;
    const float keep = 1.f - lr * t.decay;
    const bool dither = kBits == 8 && *A.step > A.nearest;
    P* const p = static_cast<P*>(t.param) + base + lane * 4;
    const G* const g = static_cast<const G*>(t.grad) + base + lane * 4;
    const long long at = t.start + base;
    const unsigned seed = static_cast<unsigned>(at / 4 + lane) * kRoot2 + static_cast<unsigned>(*A.step) * kRoot3;
    const long long left0 = t.elements - base;     // elements from the wave's first on
    if (left0 <= 0) return;
    auto run = [&](auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        Float4 pv[kBlocks], gv[kBlocks], mv[kBlocks], vv[kBlocks];
        int mc[kBlocks], vc[kBlocks];
        float ms[kBlocks], vs[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const long long left = left0 - b * kBlock - lane * 4;
            if (!kWhole && left0 <= b * kBlock) break;
            pv[b] = load<P, kWhole>(p + b * kBlock, left);
            gv[b] = load<G, kWhole>(g + b * kBlock, left);
            if constexpr (kBits == 32) {
                mv[b] = *reinterpret_cast<const Float4*>(static_cast<float*>(A.m) + at + b * kBlock + lane * 4);
                vv[b] = *reinterpret_cast<const Float4*>(static_cast<float*>(A.v) + at + b * kBlock + lane * 4);
            } else {
                mc[b] = *reinterpret_cast<const int*>(static_cast<char*>(A.m) + at + b * kBlock + lane * 4);
                vc[b] = *reinterpret_cast<const int*>(static_cast<char*>(A.v) + at + b * kBlock + lane * 4);
                ms[b] = A.m_scale[at / kBlock + b];
                vs[b] = A.v_scale[at / kBlock + b];
            }
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const long long left = left0 - b * kBlock - lane * 4;
            if (!kWhole && left0 <= b * kBlock) break;
            if constexpr (kBits == 8) {
                mv[b] = unpack(mc[b], ms[b]);
                vv[b] = unpack(vc[b], vs[b]);
                vv[b] *= vv[b];
            }
            Float4 root;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float gg = gv[b][i] * clip;
                // (each operation rounded by itself: see quantise)
                mv[b][i] = A.beta1 * mv[b][i] + A.less1 * gg;
                vv[b][i] = A.beta2 * vv[b][i] + A.less2 * gg * gg;
                root[i] = sqrtf(vv[b][i]);
                const float step = mv[b][i] * __builtin_amdgcn_rcpf(fmaf(root[i], rates.root, A.eps));
                pv[b][i] = fmaf(-rates.size, step, pv[b][i] * keep);
                if (!kWhole && i >= left) mv[b][i] = root[i] = vv[b][i] = 0.f;
            }
            store<P, kWhole>(p + b * kBlock, pv[b], left);
            if constexpr (kBits == 32) {
                *reinterpret_cast<Float4*>(static_cast<float*>(A.m) + at + b * kBlock + lane * 4) = mv[b];
                *reinterpret_cast<Float4*>(static_cast<float*>(A.v) + at + b * kBlock + lane * 4) = vv[b];
            } else {
                const unsigned bits = dither ? mixed(seed + b * (kBlock / 4) * kRoot2) : 0;
                const float m_scale = quantise<false>(mv[b], mc[b], dither, bits);
                const float v_scale = quantise<true>(root, vc[b], dither, bits);
                *reinterpret_cast<int*>(static_cast<char*>(A.m) + at + b * kBlock + lane * 4) = mc[b];
                *reinterpret_cast<int*>(static_cast<char*>(A.v) + at + b * kBlock + lane * 4) = vc[b];
                if (lane == 0) {
                    A.m_scale[at / kBlock + b] = m_scale;
                    A.v_scale[at / kBlock + b] = v_scale;
                }
            }
        }
    };
    if (left0 >= kBlocks * kBlock) run(std::true_type{});
    else run(std::false_type{});
}

template <class P, class G, int kBits>
hipError_t launch(const AdamwArgs& L, unsigned grid, hipStream_t st) {
    k_adamw<P, G, kBits><<<grid, kThreads, 0, st>>>(L);
    return hipGetLastError();
}

}  // namespace

hipError_t adamw_launch(const hx_adamw_args& A) {
    const hipStream_t st = static_cast<hipStream_t>(A.stream);
    AdamwArgs L;
    L.m = A.m, L.v = A.v, L.m_scale = A.m_scale, L.v_scale = A.v_scale;
    L.beta1 = static_cast<float>(A.beta1), L.beta2 = static_cast<float>(A.beta2);
    L.less1 = static_cast<float>(1. - A.beta1), L.less2 = static_cast<float>(1. - A.beta2);
    L.eps = static_cast<float>(A.eps), L.lr = static_cast<float>(A.lr);
    L.grad_scale = static_cast<float>(A.grad_scale);
    L.grad_scale_ptr = A.grad_scale_ptr, L.lr_ptr = A.lr_ptr;
    L.rates = reinterpret_cast<const Rates*>(A.step + 1);
    L.step = A.step, L.nearest = std::llround(1. / (1. - std::max(A.beta1, A.beta2)));
    k_count<<<1, 1, 0, st>>>(A.step, std::log(A.beta1), std::log(A.beta2), L.lr, L.lr_ptr);
    hipError_t e = hipGetLastError();
    // tensors of one pair of types share launches; none follows one that failed
    for (int64_t type = HX_F32; type <= HX_BF16; ++type)
        for (int64_t grad = HX_F32; grad <= HX_BF16; ++grad) {
            long long groups = 0;
            L.count = 0;
            auto flush = [&] {
                if (!L.count) return;
                e = with_type(type, [&](auto p) {
                    return with_type(grad, [&](auto g) {
                        using P = decltype(p);
                        using G = decltype(g);
                        return A.bits == 8 ? launch<P, G, 8>(L, static_cast<unsigned>(groups), st)
                                           : launch<P, G, 32>(L, static_cast<unsigned>(groups), st);
                    });
                });
                groups = 0;
                L.count = 0;
            };
            for (int64_t i = 0; i < A.count && e == hipSuccess; ++i) {
                const long long n = A.elements[i], more = (n + kChunk - 1) / kChunk;
                if (A.types[i] != type || A.grad_types[i] != grad || !n) continue;
                if (L.count == kTensors || groups + more > (1 << 23)) flush();
                L.tensor[L.count++] = {A.params[i], A.grads[i], n, A.starts[i], static_cast<unsigned>(groups),
                                       static_cast<float>(A.weight_decays[i])};
                groups += more;
            }
            if (e == hipSuccess) flush();
        }
    return e;
}

}  // namespace hx
