// Linear attention with a decay for each head.  Outputs and gradients are the same sum over
// different operands,
//
//   y_i = sum over j <= i of e^{g (i - j)} (a_i . b_j) c_j + (what a state brings in),
//
// with i counting steps from the sequence's first (forward) or last (reverse):
//   o:  a, b, c = q, k, v   forward, state k v^T        dq: a, b, c = do, v, k  forward, state v k^T
//   dk: a, b, c = v, do, q  reverse, state do q^T       dv: a, b, c = k, q, do  reverse, state q do^T
#include <algorithm>
#include <type_traits>

#include "readout.h"

namespace hx {
namespace {

constexpr int kThreads = 256;

// The logarithm of a decay, finite: -inf as a number whose exponential is 0 after one step, so
// that e^{g 0} stays 1.  Decays are expf(g n), made once a workgroup or once a chunk: g goes in as
// it is, and their error is that of one product and one exponential.
__device__ __forceinline__ float decay_of(float log_decay) { return log_decay < -1e4f ? -1e4f : log_decay; }

struct ScanArgs {
    const void *a, *b, *c;
    long long a_stride[3], b_stride[3], c_stride[3];
    int a_each, b_each, c_each;       // heads that share one of a, b, c: head h reads head h / each
    int heads, da, dc, time;
    bool reverse;
    float scale_in, scale_out;       // of what enters the state, and of y
    const float* log_decay;
    const int32_t* lengths;
    const float* state_in;
    float* state_out;
    int row_stride, col_stride;      // of a state's da and dc
    float* states;                   // (batch, heads, segments - 1) states: what enters segment 1, 2, ...
    void* y;
    long long y_stride[3];
    bool y_f32;                      // y is fp32 whatever the inputs are
};

// ------------------------------------------------------------------- one step
// One workgroup per (sequence, head).  Lanes lie along a state's rows, kV columns each, so that
// the state streams through as it lies in memory; k and q wait in LDS.  Bound by the state's
// bytes, read and written once: 256 x 16 states of 128 x 128, a twentieth of the rows without a
// slot (510 MB), in 96 to 101 us, 5.1 to 5.3 TB/s (a copy of 2 GiB reaches 4.8; of a pool of
// 315 MB some may stay cached from call to call).  A single row is bound by the call (11 us, 4.6
// of them on the GPU).
template <class T, int kV>
__global__ void __launch_bounds__(kThreads) k_step(ScanArgs S, float* states, const int32_t* slots, long long n_slots,
                                                   int lanes) {
    typedef float Vec __attribute__((ext_vector_type(kV)));
    constexpr int kBatch = 8;                  // rows in flight
    __shared__ float lq[kAttnMaxDim], lk[kAttnMaxDim], part[kThreads * kV];
    const int batch = blockIdx.x / S.heads, h = blockIdx.x - batch * S.heads;
    const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes, groups = kThreads / lanes;
    const int col = lane * kV;
    const long long slot = slots ? slots[batch] : batch;
    const bool run = slot >= 0 && slot < n_slots, mine = run && col < S.dc;
    T* o = static_cast<T*>(S.y) + batch * S.y_stride[0] + h * S.y_stride[2];
    float* s = states + (slot * S.heads + h) * static_cast<long long>(S.da) * S.dc + col;
    Vec x[kBatch];
    auto fetch = [&](int row0) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int row = row0 + i * groups;
            if (mine && row < S.da) x[i] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(s + row * S.dc));
        }
    };
    fetch(group);
    const float decay = expf(S.log_decay[h]);
    const T* a = static_cast<const T*>(S.a) + batch * S.a_stride[0] + (h / S.a_each) * S.a_stride[2];
    const T* b = static_cast<const T*>(S.b) + batch * S.b_stride[0] + (h / S.b_each) * S.b_stride[2];
    const T* c = static_cast<const T*>(S.c) + batch * S.c_stride[0] + (h / S.c_each) * S.c_stride[2];
    if (threadIdx.x < S.da) {
        lq[threadIdx.x] = to_f32(a[threadIdx.x]);
        lk[threadIdx.x] = to_f32(b[threadIdx.x]);
    }
    Vec v = {}, sum = {};
    if (mine)
#pragma unroll
        for (int i = 0; i < kV; ++i) v[i] = to_f32(c[col + i]);
    __syncthreads();
    for (int row0 = group; row0 < S.da; row0 += kBatch * groups) {
        if (row0 != group) fetch(row0);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int row = row0 + i * groups;
            if (mine && row < S.da) {
                const float kk = lk[row], qq = lq[row];
#pragma unroll
                for (int j = 0; j < kV; ++j) {
                    x[i][j] = fmaf(kk, v[j], x[i][j] * decay);
                    sum[j] = fmaf(qq, x[i][j], sum[j]);
                }
                __builtin_nontemporal_store(x[i], reinterpret_cast<Vec*>(s + row * S.dc));
            }
        }
    }
    *reinterpret_cast<Vec*>(part + threadIdx.x * kV) = sum;
    __syncthreads();
    if (threadIdx.x < S.dc) {
        float y = 0.f;
        for (int k = 0; k < groups; ++k) y += part[k * lanes * kV + threadIdx.x];
        o[threadIdx.x] = from_f32<T>(run ? y * S.scale_out : 0.f);
    }
}

// ------------------------------------------------------------------- whole sequences
// Chunks of kC steps.  With i, j counted inside a chunk of n steps, X the state that enters it
// and off 1 (forward) or 0 (reverse, where a state has not decayed before its first step):
//   P_ij = scale_in scale_out e^{g (i - j)} (a_i . b_j) for j <= i
//   y_i  = sum_j P_ij c_j + scale_out e^{g (i + off)} X^T a_i
//   X'   = e^{g n} X + sum_j b_j (scale_in e^{g (n - off - j)} c_j)^T
// are products of matrices.  A workgroup walks through the chunks of one (sequence, head, slice of
// c's columns, segment of the steps); each wave keeps X^T's rows for its own columns in
// accumulator registers, whose layout (lane: one column, four rows) is at the same time that of
// an operand, so X enters y's product without leaving the registers.  y and P are made transposed
// for the same reason: P goes to LDS, and y to memory, four neighbours a lane.
//
// No step's output looks at a later step: P over the diagonal is made zero, not multiplied by it,
// and a chunk ends before a step whose c holds an infinity or a NaN (zero times that is NaN),
// unless that is its first.  An input of nothing but NaN makes every step a chunk.
//
// Few sequences are cut into segments: their own states first (from zero, in a launch that reads
// b and c alone), joined one after another, then every segment with the state that enters it.
// The price is b and c read twice.
//
// What bounds it, bf16, 65536 steps of 8 heads of 128 x 128 (537 MB, 113 us at a copy's rate):
// 236 us, of which about 66 for the segments' states (4 TB/s), 15 to join them and 155 for the
// rest, in which a wave issues 3200 cycles of matrix and 3300 of other vector instructions a chunk
// of its 16,900, two waves a SIMD: neither memory nor matrix cores are full, barriers and LDS reads
// lie between.  Short sequences are chains of chunks, 4 to 8 us each (777 steps of 13 x 12 sequences
// and heads, 96 x 80 in fp16: 29, 6 and 65 us).  fp32 matrix instructions take 16 times as long:
// there they bound it.  Sizes that are no whole number of pieces load and store element by element,
// and some of their kernels spill (36 to 304 bytes a lane; 128 x 128 in bf16: 156).
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Reduction indices are taken 32 at a time, eight a lane; which eight is free as long as both
// operands agree, and is chosen so that every LDS access is whole and without bank conflicts
// (two reads of 8 bytes where one of 16 does: 2400 of 4500 LDS cycles a chunk were conflicts).
//
// bf16 inputs: 32 indices an instruction.  Products of inputs are exact in fp32; P and the
// state as it enters y (Sum) are two bf16 terms, good to 2^-17, so that the only rounding of y
// that counts is its own.  The state itself stays fp32: its weighted c enters as three bf16
// terms (24 bits).
struct MathBf16 {
    using Elem = __bf16;
    using Raw = bf16x8;
    using Frag = bf16x4;
    using Pair = bf16x8;
    using Term = bf16x4;
    struct Sum {
        bf16x4 h, l;
    };
    struct SumPair {
        bf16x8 h, l;
    };
    static constexpr int kC = 64, kPiece = 8, kPlanes = 1, kPlanesP = 2, kTerms = 3;
    static constexpr int kPadA = 8, kPadB = 0, kPadC = 16, kPadP = 8;
    static __device__ __forceinline__ f32x4 mma(f32x4 acc, Pair a, Pair b) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ Frag frag(f32x4 x) { return __builtin_convertvector(x, Frag); }
    // (from the packed bits: converted one by one, the numbers are rounded once more for it)
    static __device__ __forceinline__ f32x4 wide(Frag x) {
        typedef unsigned Two __attribute__((ext_vector_type(2)));
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const Two u = __builtin_bit_cast(Two, x);
        const f32x2 even = __builtin_bit_cast(f32x2, u << 16), odd = __builtin_bit_cast(f32x2, u & 0xffff0000u);
        return f32x4{even[0], odd[0], even[1], odd[1]};
    }
    static __device__ __forceinline__ Pair pair(Frag a, Frag b) {
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    static __device__ __forceinline__ Sum sum(f32x4 x) {
        const Frag h = frag(x);
        return {h, frag(x - wide(h))};
    }
    static __device__ __forceinline__ SumPair sum_pair(Sum a, Sum b) { return {pair(a.h, b.h), pair(a.l, b.l)}; }
    static __device__ __forceinline__ f32x4 mma_sum(f32x4 acc, SumPair x, Pair a) { return mma(mma(acc, x.l, a), x.h, a); }
    static __device__ __forceinline__ f32x4 mma_by_sum(f32x4 acc, Pair c, SumPair p) { return mma(mma(acc, c, p.l), c, p.h); }
    // b times weighted c in terms
    static __device__ __forceinline__ Term term(f32x4 x) { return frag(x); }
    static __device__ __forceinline__ f32x4 wide_term(Term x) { return wide(x); }
    static __device__ __forceinline__ f32x4 mma_terms(f32x4 acc, Pair b, const Term (&w0)[kTerms], const Term (&w1)[kTerms]) {
#pragma unroll
        for (int t = 0; t < kTerms; ++t) acc = mma(acc, b, pair(w0[t], w1[t]));
        return acc;
    }
    // pieces and fragments to LDS (arrays of several planes: kPlane from one to the next)
    template <int kPlane>
    static __device__ __forceinline__ void store(Elem* at, Raw x) { *reinterpret_cast<Raw*>(at) = x; }
    template <int kPlane>
    static __device__ __forceinline__ void store_sum(Elem* at, Sum x) {
        *reinterpret_cast<Frag*>(at) = x.h;
        *reinterpret_cast<Frag*>(at + kPlane) = x.l;
    }
    // State row (a's and b's column) that accumulator rows g4 .. + 3 of tile rt hold: tiles 2K and
    // 2K + 1 take turns of four in 32 columns, so that a lane's eight are neighbours in a.
    static __device__ __forceinline__ int row(int rt, int g4) { return rt / 2 * 32 + g4 * 2 + rt % 2 * 4; }
    // a in rows: eight neighbours, against the state; or the eight that lie together in b, against b.
    template <int kPlane>
    static __device__ __forceinline__ Pair a_pair(const Elem* row, int k, int g4) {
        return *reinterpret_cast<const Pair*>(row + k * 32 + g4 * 2);
    }
    template <int kPlane>
    static __device__ __forceinline__ Pair a_like_b(const Elem* row, int k, int g4) {
        const Elem* at = row + k * 32 + g4 / 4 % 2 * 16 + g4 / 8 * 4;
        return pair(*reinterpret_cast<const Frag*>(at), *reinterpret_cast<const Frag*>(at + 8));
    }
    // b is read by rows and by columns: of each 32 columns first tile 2K's, then tile 2K + 1's, and
    // the 16-byte slots of a row exchanged by an exclusive or with f(row), which differs for 16 rows
    // and, without its lowest bit, for eight.
    template <int kDA>
    static __device__ __forceinline__ int b_at(int row, int place) {
        constexpr int kSlots = kDA / 8 < 16 ? kDA / 8 : 16, kPer = 16 / kSlots;
        const int q = row % 16 / kPer;
        const int f = (q * 2 & (kSlots - 1)) | q / (kSlots / 2);
        return row * kDA + ((place / 8 ^ f) * 8) + place % 8;
    }
    template <int kDA>
    static __device__ __forceinline__ Pair b_pair(const Elem* lb, int row, int k, int g4) {
        return *reinterpret_cast<const Pair*>(lb + b_at<kDA>(row, k * 32 + g4 * 2));
    }
    template <int kDA>
    static __device__ __forceinline__ void b_store(Elem* lb, int row, int col, Pair x) {
        const int place = col / 32 * 32 + col % 32 / 2;
        *reinterpret_cast<Frag*>(lb + b_at<kDA>(row, place)) = __builtin_shufflevector(x, x, 0, 1, 2, 3);
        *reinterpret_cast<Frag*>(lb + b_at<kDA>(row, place + 16)) = __builtin_shufflevector(x, x, 4, 5, 6, 7);
    }
    // Column `lane % 16` of a 16 x 16 block, rows 4 (lane / 16) .. + 3: the transposing read takes
    // four neighbours of row (lane % 16) / 4 from each lane.
    static __device__ __forceinline__ Frag turned(const Elem* at) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) Frag*)at);
    }
    template <int kDA>
    static __device__ __forceinline__ Frag b_column(const Elem* lb, int sb, int rt, int lane) {
        return turned(lb + b_at<kDA>(sb * 16 + 4 * (lane / 16) + lane % 16 / 4, rt * 16 + 4 * (lane % 4)));
    }
    template <int kPlane>
    static __device__ __forceinline__ Frag c_column(const Elem* lc, int stride, int sb, int col, int lane) {
        return turned(lc + (sb * 16 + 4 * (lane / 16) + lane % 16 / 4) * stride + col + 4 * (lane % 4));
    }
    // P's columns in the order that c's column fragments have
    static __device__ __forceinline__ int p_at(int sb, int g4) { return sb / 2 * 32 + g4 * 2 + sb % 2 * 4; }
    template <int kPlane>
    static __device__ __forceinline__ SumPair p_pair(const Elem* row, int sb, int g4) {
        return {*reinterpret_cast<const Pair*>(row + p_at(sb, g4)), *reinterpret_cast<const Pair*>(row + kPlane + p_at(sb, g4))};
    }
};

// fp16 inputs: each exactly the sum of two bf16 numbers (8 and 3 bits; fp16 itself has not the
// range that P and states need), held in LDS as two planes.  P and the state as it enters y are
// two bf16 terms as they are for bf16; of four products of terms the three larger ones are made, five
// of six in the state's update, which misses 2^-25 (13 x 777 steps, 12 heads of 96 x 80: 95 us; with
// fp32 instructions 117).  An infinite input gives NaN where it would give infinity.
struct MathF16 {
    using One = MathBf16;
    using Elem = __bf16;
    using Raw = f16x8;
    struct Frag {
        bf16x4 h, l;
    };
    struct Pair {
        bf16x8 h, l;
    };
    using Term = bf16x4;
    using Sum = One::Sum;
    using SumPair = One::SumPair;
    static constexpr int kC = 32, kPiece = 8, kPlanes = 2, kPlanesP = 2, kTerms = 3;
    static constexpr int kPadA = One::kPadA, kPadB = One::kPadB, kPadC = One::kPadC, kPadP = One::kPadP;
    static __device__ __forceinline__ f32x4 mma(f32x4 acc, Pair a, Pair b) {
        return One::mma(One::mma(One::mma(acc, a.h, b.l), a.l, b.h), a.h, b.h);
    }
    static __device__ __forceinline__ Sum sum(f32x4 x) { return One::sum(x); }
    static __device__ __forceinline__ SumPair sum_pair(Sum a, Sum b) { return One::sum_pair(a, b); }
    static __device__ __forceinline__ f32x4 mma_sum(f32x4 acc, SumPair x, Pair a) { return mma(acc, {x.h, x.l}, a); }
    static __device__ __forceinline__ f32x4 mma_by_sum(f32x4 acc, Pair c, SumPair p) { return mma(acc, c, {p.h, p.l}); }
    static __device__ __forceinline__ f32x4 wide(Frag x) { return One::wide(x.h) + One::wide(x.l); }
    static __device__ __forceinline__ Pair pair(Frag a, Frag b) { return {One::pair(a.h, b.h), One::pair(a.l, b.l)}; }
    static __device__ __forceinline__ Term term(f32x4 x) { return One::frag(x); }
    static __device__ __forceinline__ f32x4 wide_term(Term x) { return One::wide(x); }
    static __device__ __forceinline__ f32x4 mma_terms(f32x4 acc, Pair b, const Term (&w0)[kTerms], const Term (&w1)[kTerms]) {
#pragma unroll
        for (int t = kTerms - 1; t >= 0; --t) {
            const bf16x8 w = One::pair(w0[t], w1[t]);
            if (t < kTerms - 1) acc = One::mma(acc, b.l, w);
            acc = One::mma(acc, b.h, w);
        }
        return acc;
    }
    static __device__ __forceinline__ Pair split(Raw x) {
        typedef float f32x8 __attribute__((ext_vector_type(8)));
        const f32x8 w = __builtin_convertvector(x, f32x8);
        const SumPair p = One::sum_pair(One::sum(w.lo), One::sum(w.hi));
        return {p.h, p.l};
    }
    template <int kPlane>
    static __device__ __forceinline__ void store(Elem* at, Raw x) {
        const Pair p = split(x);
        One::store<0>(at, p.h), One::store<0>(at + kPlane, p.l);
    }
    template <int kPlane>
    static __device__ __forceinline__ void store_sum(Elem* at, Sum x) { One::store_sum<kPlane>(at, x); }
    static __device__ __forceinline__ int row(int rt, int g4) { return One::row(rt, g4); }
    template <int kPlane>
    static __device__ __forceinline__ Pair a_pair(const Elem* row, int k, int g4) {
        return {One::a_pair<0>(row, k, g4), One::a_pair<0>(row + kPlane, k, g4)};
    }
    template <int kPlane>
    static __device__ __forceinline__ Pair a_like_b(const Elem* row, int k, int g4) {
        return {One::a_like_b<0>(row, k, g4), One::a_like_b<0>(row + kPlane, k, g4)};
    }
    template <int kDA>
    static __device__ __forceinline__ Pair b_pair(const Elem* lb, int row, int k, int g4) {
        return {One::b_pair<kDA>(lb, row, k, g4), One::b_pair<kDA>(lb + kC * kDA, row, k, g4)};
    }
    template <int kDA>
    static __device__ __forceinline__ void b_store(Elem* lb, int row, int col, Raw x) {
        const Pair p = split(x);
        One::b_store<kDA>(lb, row, col, p.h), One::b_store<kDA>(lb + kC * kDA, row, col, p.l);
    }
    template <int kDA>
    static __device__ __forceinline__ Frag b_column(const Elem* lb, int sb, int rt, int lane) {
        return {One::b_column<kDA>(lb, sb, rt, lane), One::b_column<kDA>(lb + kC * kDA, sb, rt, lane)};
    }
    template <int kPlane>
    static __device__ __forceinline__ Frag c_column(const Elem* lc, int stride, int sb, int col, int lane) {
        return {One::c_column<0>(lc, stride, sb, col, lane), One::c_column<0>(lc + kPlane, stride, sb, col, lane)};
    }
    static __device__ __forceinline__ int p_at(int sb, int g4) { return One::p_at(sb, g4); }
    template <int kPlane>
    static __device__ __forceinline__ SumPair p_pair(const Elem* row, int sb, int g4) { return One::p_pair<kPlane>(row, sb, g4); }
};

// fp32 inputs, in fp32 throughout.
struct MathF32 {
    using Elem = float;
    using Raw = f32x4;
    using Frag = f32x4;
    struct Pair {
        f32x4 x[2];
    };
    using Term = f32x4;
    using Sum = f32x4;
    using SumPair = Pair;
    static constexpr int kC = 32, kPiece = 4, kPlanes = 1, kPlanesP = 1, kTerms = 1;
    static constexpr int kPadA = 4, kPadB = 4, kPadC = 4, kPadP = 4;
    static __device__ __forceinline__ f32x4 mma(f32x4 acc, Pair a, Pair b) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x[h][i], b.x[h][i], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ f32x4 wide(Frag x) { return x; }
    static __device__ __forceinline__ Pair pair(Frag a, Frag b) { return {a, b}; }
    static __device__ __forceinline__ Sum sum(f32x4 x) { return x; }
    static __device__ __forceinline__ SumPair sum_pair(Sum a, Sum b) { return {a, b}; }
    static __device__ __forceinline__ f32x4 mma_sum(f32x4 acc, SumPair x, Pair a) { return mma(acc, x, a); }
    static __device__ __forceinline__ f32x4 mma_by_sum(f32x4 acc, Pair c, SumPair p) { return mma(acc, c, p); }
    static __device__ __forceinline__ Term term(f32x4 x) { return x; }
    static __device__ __forceinline__ f32x4 wide_term(Term x) { return x; }
    static __device__ __forceinline__ f32x4 mma_terms(f32x4 acc, Pair b, const Term (&w0)[kTerms], const Term (&w1)[kTerms]) {
        return mma(acc, b, pair(w0[0], w1[0]));
    }
    template <int kPlane>
    static __device__ __forceinline__ void store(Elem* at, Raw x) { *reinterpret_cast<Raw*>(at) = x; }
    template <int kPlane>
    static __device__ __forceinline__ void store_sum(Elem* at, Sum x) { *reinterpret_cast<Frag*>(at) = x; }
    static __device__ __forceinline__ int row(int rt, int g4) { return rt * 16 + g4; }
    template <int kPlane>
    static __device__ __forceinline__ Pair a_pair(const Elem* row, int k, int g4) {
        return {*reinterpret_cast<const Frag*>(row + k * 32 + g4), *reinterpret_cast<const Frag*>(row + k * 32 + 16 + g4)};
    }
    template <int kPlane>
    static __device__ __forceinline__ Pair a_like_b(const Elem* row, int k, int g4) { return a_pair<0>(row, k, g4); }
    template <int kDA>
    static __device__ __forceinline__ Pair b_pair(const Elem* lb, int row, int k, int g4) {
        return a_pair<0>(lb + row * (kDA + kPadB), k, g4);
    }
    template <int kDA>
    static __device__ __forceinline__ void b_store(Elem* lb, int row, int col, Frag x) {
        *reinterpret_cast<Frag*>(lb + row * (kDA + kPadB) + col) = x;
    }
    template <int kPlane>
    static __device__ __forceinline__ Frag c_column(const Elem* lc, int stride, int sb, int col, int lane) {
        const Elem* at = lc + (sb * 16 + 4 * (lane / 16)) * stride + col + lane % 16;
        return Frag{at[0], at[stride], at[2 * stride], at[3 * stride]};
    }
    template <int kDA>
    static __device__ __forceinline__ Frag b_column(const Elem* lb, int sb, int rt, int lane) {
        return c_column<0>(lb, kDA + kPadB, sb, rt * 16, lane);
    }
    static __device__ __forceinline__ int p_at(int sb, int g4) { return sb * 16 + g4; }
    template <int kPlane>
    static __device__ __forceinline__ Pair p_pair(const Elem* row, int sb, int g4) {
        return {*reinterpret_cast<const Frag*>(row + sb * 16 + g4),
                *reinterpret_cast<const Frag*>(row + sb * 16 + 16 + g4)};
    }
};

// The products' mathematics, the input's type and four of them, the exponent's bits and lowest bit
// of the numbers in 32 bits.
template <class T> struct InputOf;
template <> struct InputOf<float> {
    static constexpr int kType = HX_F32;
    static constexpr unsigned kExponent = 0x7f800000u, kUnit = 0x00800000u;
    using Math = MathF32;
    using Elem = float;
    using Four = f32x4;
};
template <> struct InputOf<__half> {
    static constexpr int kType = HX_F16;
    static constexpr unsigned kExponent = 0x7c007c00u, kUnit = 0x04000400u;
    using Math = MathF16;
    using Elem = _Float16;
    using Four = f16x4;
};
template <> struct InputOf<__hip_bfloat16> {
    static constexpr int kType = HX_BF16;
    static constexpr unsigned kExponent = 0x7f807f80u, kUnit = 0x00800080u;
    using Math = MathBf16;
    using Elem = __bf16;
    using Four = bf16x4;
};

// Rows [0, n) of a chunk into registers, kD columns padded with zeros, R rows a round of the
// workgroup.  kWhole: d is a whole number of pieces and a round's rows are within 2 GiB, so that
// a load is one instruction with a uniform address and the same 32-bit offset in every round
// (64-bit addresses by lane, twelve a thread, went to scratch memory and were waited for one by
// one).  The choice is the kernel's: a register that either of two loads may fill is waited for
// at once.  Pieces start at any element: loads need no alignment.
template <class T, int kD, int kT, bool kWhole>
struct Tile {
    using In = InputOf<T>;
    using Math = typename In::Math;
    static constexpr int kP = Math::kPiece, kRowPieces = kD / kP, kRows = kT / kRowPieces;
    static constexpr int kN = kRows < Math::kC ? Math::kC / kRows : 1;
    static_assert(kRows * kRowPieces == kT && (kN * kRows == Math::kC || kN == 1), "whole rounds of rows");
    typedef typename Math::Raw Raw;
    typedef Raw Any __attribute__((aligned(sizeof(T))));
    Raw raw[kN];
    const T* base;          // row 0 of the sequence (reverse: row R - 1 of a round that starts there)
    long long step;         // from row to row
    int row, col, d;        // of this thread in a round
    unsigned offset;        // bytes

    __device__ __forceinline__ void start(const T* p, long long stride, bool reverse, int columns) {
        row = threadIdx.x / kRowPieces, col = threadIdx.x % kRowPieces * kP, d = columns;
        step = reverse ? -stride : stride;
        if constexpr (kWhole) {
            base = reverse ? p - (kRows - 1) * stride : p;
            offset = static_cast<unsigned>(((reverse ? kRows - 1 - row : row) * stride + col) * sizeof(T));
            if (col >= d) row = Math::kC;      // no row has these columns
        } else {
            base = p;
        }
    }
    __device__ __forceinline__ void load(long long first, int n) {       // from row `first` (in memory order) on
        // new to the compiler in every chunk, or it keeps a running 64-bit address a load by lane
        if constexpr (kWhole) asm volatile("" : "+v"(offset));
#pragma unroll
        for (int p = 0; p < kN; ++p) {
            Raw x = {};
            if constexpr (kWhole) {
                const char* at = reinterpret_cast<const char*>(base + first + p * kRows * step);
                if (row < n - p * kRows) x = *reinterpret_cast<const Any*>(at + offset);
            } else if (row + p * kRows < n) {
                const typename In::Elem* at =
                    reinterpret_cast<const typename In::Elem*>(base) + first + (row + p * kRows) * step + col;
#pragma unroll
                for (int k = 0; k < kP; ++k)
                    if (col + k < d) x[k] = at[k];
            }
            raw[p] = x;
        }
    }
    // put(row, column, piece) for the pieces of this thread
    template <class F>
    __device__ __forceinline__ void store(F put, int thread = threadIdx.x) const {
        const int i = thread / kRowPieces, j = thread % kRowPieces * kP;
#pragma unroll
        for (int p = 0; p < kN; ++p)
            if (kRows <= Math::kC || i < Math::kC) put(i + p * kRows, j, raw[p]);
    }
    // Whether an infinity or a NaN is among the pieces (their exponents are nothing but ones, and one
    // more of their lowest bit passes on).
    static __device__ __forceinline__ unsigned exponents(Raw x) {
        typedef unsigned Words __attribute__((ext_vector_type(4)));
        const Words w = (__builtin_bit_cast(Words, x) & In::kExponent) + In::kUnit;
        return w[0] | w[1] | w[2] | w[3];
    }
    static constexpr unsigned kOdd = In::kExponent + In::kUnit;
    __device__ __forceinline__ bool odd() const {
        unsigned any = 0;
#pragma unroll
        for (int p = 0; p < kN; ++p) any |= exponents(raw[p]);
        return (any & kOdd) != 0;
    }
    // f(row) for the pieces with one among them
    template <class F>
    __device__ __forceinline__ void each_odd(F f) const {
#pragma unroll
        for (int p = 0; p < kN; ++p)
            if ((exponents(raw[p]) & kOdd) != 0) f(static_cast<int>(threadIdx.x) / kRowPieces + p * kRows);
    }
};

constexpr int kJobs = 3;               // sums of one launch: the gradients are three
struct ChunkArgs {
    ScanArgs job[kJobs];
    int jobs, nslice, nseg, seg_steps; // seg_steps a multiple of the chunk
};

// A job where it lies among the kernel's arguments (indexed as a value, the array
// would be copied to every lane's scratch memory first: 157 -> 452 us).
typedef const __attribute__((address_space(4))) ScanArgs JobArgs;
__device__ __forceinline__ JobArgs& job_of(int job) {
    typedef const __attribute__((address_space(4))) ChunkArgs Args;
    return ((Args*)__builtin_amdgcn_kernarg_segment_ptr())->job[job];
}

// Four neighbours of a row to base[at], of which `columns` are there.
template <class V> using Global = __attribute__((address_space(1))) V;
template <class Out, class Four, bool kWhole, class At>
__device__ __forceinline__ void put(Global<Out>* base, At at, int columns, f32x4 v) {
    const Four w = __builtin_convertvector(v, Four);
    if constexpr (kWhole) {
        typedef Four Any __attribute__((aligned(sizeof(Out))));
        if (columns > 0) *(Global<Any>*)(base + at) = w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k < columns) base[at + k] = w[k];
    }
}

// kDA: rows of the state (a's and b's columns) padded; kW waves of kCT 16-column tiles each.
// kFull: the state fills its padding; else products of nothing but padding are left out (96 x 80
// of 128 x 128 is half the work), at the price of branches between the others.
// kStates: only the own state, from zero, of each segment but the last.
// Waves a SIMD.  Small states in chunks of 32 steps leave registers for four (2 x 4000 steps of 8 heads,
// 33 x 47, with gradient: 153 us in fp16 and fp32, with three 171 and 163).
template <class T, int kDA, int kW, int kCT>
constexpr int kWavesASimd =
    kW == 8 || (kW == 4 && kCT == 1 && kDA <= 64 && InputOf<T>::Math::kC == 32) ? 4 : 2;

template <class T, int kDA, int kW, int kCT, bool kWhole, bool kFull, bool kStates>
__global__ void __launch_bounds__(kW * 64, (kWavesASimd<T, kDA, kW, kCT>)) k_chunk(ChunkArgs A) {
    using In = InputOf<T>;
    using M = typename In::Math;
    using Elem = typename M::Elem;
    using Frag = typename M::Frag;
    constexpr int kC = M::kC, kB = kC / 16, kT = kW * 64, kDC = kW * kCT * 16, kRT = kDA / 16;
    using Pair = typename M::Pair;
    using Raw = typename M::Raw;
    constexpr int kSA = kDA + M::kPadA, kSB = kDA + M::kPadB, kSC = kDC + M::kPadC, kSP = kC + M::kPadP, kK = kRT / 2;
    constexpr int kPlaneA = kC * kSA, kPlaneC = kC * kSC, kPlaneP = kC * kSP, kPlanes = M::kPlanes;
    __shared__ __attribute__((aligned(16))) Elem la[kStates ? 1 : kPlaneA * kPlanes], lb[kC * kSB * kPlanes],
        lc[kPlaneC * kPlanes], lp[kStates ? 1 : kPlaneP * M::kPlanesP];
    // the chunk's decays, made once: of P's blocks tb - sb + 1 blocks under the diagonal (the first:
    // over it) as a lane holds them, NaN for later steps; of the entering state; of what enters at a step
    __shared__ f32x4 lfactor[kStates ? 1 : (kB + 1) * 64], lleft[kC / 4];
    __shared__ float lsince[kStates ? 1 : kC];
    __shared__ int lodd;                                   // the first step but 0 whose c is not finite
    // neighbouring workgroups take the jobs of one segment, which read much the same
    const JobArgs& S = job_of(blockIdx.x % A.jobs);
    const int lane = threadIdx.x % 64, r = lane % 16, g4 = lane / 16 * 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int part = blockIdx.x / A.jobs, slice = part % A.nslice, unit = part / A.nslice;
    const int nseg = kStates ? A.nseg - 1 : A.nseg;
    const int seg = unit % nseg, bh = unit / nseg;
    const int batch = bh / S.heads, h = bh - batch * S.heads;
    const int len = S.lengths ? min(max(S.lengths[batch], 0), S.time) : S.time;
    const int col0 = slice * kDC;                          // of the slice
    const int mine = wave * kCT * 16;                      // of the wave, in the slice
    const float g = decay_of(S.log_decay[h]);
    const int off = S.reverse ? 0 : 1;
    const float scale = S.scale_in * S.scale_out;
    const int dc_here = min(S.dc - col0, kDC);

    const T* a0 = static_cast<const T*>(S.a) + batch * S.a_stride[0] + (h / S.a_each) * S.a_stride[2];
    const T* b0 = static_cast<const T*>(S.b) + batch * S.b_stride[0] + (h / S.b_each) * S.b_stride[2];
    const T* c0 =
        static_cast<const T*>(S.c) + batch * S.c_stride[0] + (h / S.c_each) * S.c_stride[2] + col0;
    const int begin = seg * A.seg_steps, end = min(begin + A.seg_steps, S.time), stop = min(end, len);

    Tile<T, kDA, kT, kWhole> ta, tb;
    Tile<T, kDC, kT, kWhole> tc;
    if constexpr (!kStates) ta.start(a0, S.a_stride[1], S.reverse, S.da);
    tb.start(b0, S.b_stride[1], S.reverse, S.da);
    tc.start(c0, S.c_stride[1], S.reverse, dc_here);
    // in two parts: all at once, the pieces would take registers from the products beside them
    auto fetch = [&](int i0, int part) {
        const int n = min(kC, stop - i0);
        const long long t0 = S.reverse ? len - 1 - i0 : i0;
        if (part == 0) {
            if constexpr (!kStates) ta.load(t0 * S.a_stride[1], n);
            tc.load(t0 * S.c_stride[1], n);
        } else {
            tb.load(t0 * S.b_stride[1], n);
        }
    };
    fetch(begin, 0);
    fetch(begin, 1);

    // The state that enters: what came before the sequence, and the segments before this one.
    f32x4 X[kRT][kCT];
#pragma unroll
    for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
        for (int ct = 0; ct < kCT; ++ct) X[rt][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    const long long state_size = static_cast<long long>(S.da) * S.dc;
    // X at each place becomes f(X there, where that lies in a state)
    auto each_place = [&](auto f) {
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
            for (int ct = 0; ct < kCT; ++ct)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = M::row(rt, g4) + i, col = col0 + mine + ct * 16 + r;
                    if (row < S.da && col < S.dc)
                        X[rt][ct][i] = f(X[rt][ct][i], row * S.row_stride + col * S.col_stride);
                }
    };
    if constexpr (!kStates) {
        if (seg > 0) {
            const float* w = S.states + (static_cast<long long>(bh) * (A.nseg - 1) + seg - 1) * state_size;
            each_place([&](float, int at) { return w[at]; });
        }
        if (S.state_in) {
            const float left = expf(g * static_cast<float>(min(begin, len)));
            const float* w = S.state_in + bh * state_size;
            each_place([&](float x, int at) { return x + left * w[at]; });
        }
    }
    // scale_in e^{g (n - off - j)}: what is left at the chunk's end of what enters at step j
    auto make_left = [&](int n) {
        if (threadIdx.x < kC / 4) {
            f32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = threadIdx.x * 4 + i;
                w[i] = j < n ? S.scale_in * expf(g * static_cast<float>(n - off - j)) : 0.f;
            }
            lleft[threadIdx.x] = w;
        }
    };
    make_left(kC);
    int left_of = kC;                                      // the steps that lleft is made for
    if (threadIdx.x == 0) lodd = kC;
    if constexpr (!kStates) {
        for (int e = threadIdx.x; e < (kB + 1) * 64; e += kT) {
            f32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int ago = (e / 64 - 1) * 16 + r - g4 - i;
                w[i] = e >= 64 && ago >= 0 ? scale * expf(g * static_cast<float>(ago)) : __builtin_nanf("");
            }
            lfactor[e] = w;
        }
        if (threadIdx.x < kC) lsince[threadIdx.x] = S.scale_out * expf(g * static_cast<float>(threadIdx.x + off));
    }
    long long y_step = S.y_stride[1];
    unsigned long long y_base = reinterpret_cast<unsigned long long>(S.y) +
                                (batch * S.y_stride[0] + h * S.y_stride[2] + col0 + mine) * (S.y_f32 ? 4 : sizeof(T));
    asm volatile("" : "+s"(y_base), "+s"(y_step));         // held, not read from the arguments at every store
    const std::conditional_t<kWhole, unsigned, long long> y_lane = (S.reverse ? 15 - r : r) * y_step + g4;

    for (int i0 = begin, n; i0 < stop; i0 += n) {
        n = min(kC, stop - i0);
        __syncthreads();                       // the chunk before is done with
        if (n != left_of) make_left(left_of = n);
        if constexpr (!kStates)
            ta.store([&](int i, int col, Raw x) { M::template store<kPlaneA>(la + i * kSA + col, x); });
        tb.store([&](int i, int col, Raw x) { M::template b_store<kDA>(lb, i, col, x); });
        tc.store([&](int i, int col, Raw x) { M::template store<kPlaneC>(lc + i * kSC + col, x); });
        if constexpr (!kStates)
            if (tc.odd())
                tc.each_odd([&](int i) {
                    if (i > 0) atomicMin(&lodd, i);
                });
        __syncthreads();
        // whether columns 32 k .. of a and b are there, and the wave's column tile ct
        auto there = [&](int k) { return kFull || k * 32 < S.da; };
        auto column = [&](int ct) { return kFull || col0 + mine + ct * 16 < S.dc; };
        Frag c[kB][kCT];
        if constexpr (!kStates) {
            const int first_odd = lodd;
            // P's blocks, as many for each wave
            constexpr int kEach = kB * kB > kW ? kB * kB / kW : 1;
            static_assert((kEach * kW == kB * kB || kEach == 1) && (kEach % kB == 0 || kB % kEach == 0),
                          "whole rows or parts of one");
            const int block0 = wave * kEach;
            if (kEach * kW == kB * kB || block0 < kB * kB) {
                f32x4 p[kEach];
#pragma unroll
                for (int e = 0; e < kEach; ++e) p[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kK; ++k)
                    if (there(k)) {
                        Pair pa;
#pragma unroll
                        for (int e = 0; e < kEach; ++e) {
                            if (e % kB == 0) pa = M::template a_like_b<kPlaneA>(la + ((block0 + e) / kB * 16 + r) * kSA, k, g4);
                            p[e] = M::mma(p[e], M::template b_pair<kDA>(lb, (block0 + e) % kB * 16 + r, k, g4), pa);
                        }
                    }
                // lane: step tb*16 + r, earlier steps sb*16 + g4 .. + 3
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int tb_ = (block0 + e) / kB, sb = (block0 + e) % kB;
                    const f32x4 w = lfactor[(max(tb_ - sb, -1) + 1) * 64 + lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[e][i] = w[i] == w[i] ? p[e][i] * w[i] : 0.f;
                    M::template store_sum<kPlaneP>(lp + (tb_ * 16 + r) * kSP + M::p_at(sb, g4), M::sum(p[e]));
                }
            }
            // (P is made with the steps that this takes out: in the rows that stay it is zero there)
            const int odd = __builtin_amdgcn_readfirstlane(first_odd);
            if (odd < n) {
                n = odd;
                __syncthreads();               // all have read it
                if (threadIdx.x == 0) lodd = kC;
                make_left(left_of = n);
                int thread = threadIdx.x;
                asm volatile("" : "+v"(thread));       // its addresses are made here, not kept
                tb.store([&](int i, int col, Raw) {
                    if (i >= n) M::template b_store<kDA>(lb, i, col, Raw{});
                }, thread);
                tc.store([&](int i, int col, Raw) {
                    if (i >= n) M::template store<kPlaneC>(lc + i * kSC + col, Raw{});
                }, thread);
                __syncthreads();
            }
        }
#pragma unroll
        for (int sb = 0; sb < kB; ++sb)
#pragma unroll
            for (int ct = 0; ct < kCT; ++ct) c[sb][ct] = M::template c_column<kPlaneC>(lc, kSC, sb, mine + ct * 16, lane);
        if constexpr (!kStates) {
            __syncthreads();                   // P is whole
            // all blocks of steps at a time, so that the state's terms are made once and not kept: what
            // the entering state adds, then the chunk's own steps
            if (column(0)) {
                f32x4 y[kB][kCT];
#pragma unroll
                for (int t = 0; t < kB; ++t)
#pragma unroll
                    for (int ct = 0; ct < kCT; ++ct) y[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < kK; ++k)
                    if (there(k)) {
                        Pair pa[kB];
#pragma unroll
                        for (int t = 0; t < kB; ++t) pa[t] = M::template a_pair<kPlaneA>(la + (t * 16 + r) * kSA, k, g4);
#pragma unroll
                        for (int ct = 0; ct < kCT; ++ct) {
                            const typename M::SumPair x = M::sum_pair(M::sum(X[2 * k][ct]), M::sum(X[2 * k + 1][ct]));
#pragma unroll
                            for (int t = 0; t < kB; ++t) y[t][ct] = M::mma_sum(y[t][ct], x, pa[t]);
                        }
                    }
#pragma unroll
                for (int t = 0; t < kB; ++t) {
                    const float since = lsince[t * 16 + r];
#pragma unroll
                    for (int ct = 0; ct < kCT; ++ct) y[t][ct] *= since;
#pragma unroll
                    for (int sb = 0; sb <= t; sb += 2) {
                        const typename M::SumPair pp = M::template p_pair<kPlaneP>(lp + (t * 16 + r) * kSP, sb, g4);
#pragma unroll
                        for (int ct = 0; ct < kCT; ++ct)
                            y[t][ct] = M::mma_by_sum(y[t][ct], M::pair(c[sb][ct], c[sb + 1][ct]), pp);
                    }
                    // lane: step t*16 + r, columns g4 .. + 3 of each tile
                    const int i1 = i0 + t * 16;
                    const long long at = (S.reverse ? len - 1 - i1 - 15 : i1) * y_step;     // of the least step
                    if (t * 16 + r < n) {
#pragma unroll
                        for (int ct = 0; ct < kCT; ++ct) {
                            const int columns = S.dc - (col0 + mine + ct * 16 + g4);
                            if (S.y_f32)
                                put<float, f32x4, kWhole>((Global<float>*)y_base + at + ct * 16, y_lane,
                                                          columns, y[t][ct]);
                            else
                                put<typename In::Elem, typename In::Four, kWhole>(
                                    (Global<typename In::Elem>*)y_base + at + ct * 16, y_lane, columns,
                                    y[t][ct]);
                        }
                    }
                }
            }
        }
        if (i0 + n < stop) fetch(i0 + n, 0);
        // the state that leaves
        const float keep = expf(g * static_cast<float>(n));
#pragma unroll
        for (int rt = 0; rt < kRT; ++rt)
#pragma unroll
            for (int ct = 0; ct < kCT; ++ct) X[rt][ct] *= keep;
#pragma unroll
        for (int sb = 0; sb < kB; sb += 2) {
            if (sb == kB - 2 && i0 + n < stop) fetch(i0 + n, 1);
            if (!column(0)) continue;
            typename M::Term wc[2][kCT][M::kTerms];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const f32x4 w0 = lleft[(sb + e) * 4 + g4 / 4];
#pragma unroll
                for (int ct = 0; ct < kCT; ++ct) {
                    f32x4 w = M::wide(c[sb + e][ct]) * w0;
#pragma unroll
                    for (int k = 0; k < M::kTerms; ++k) {
                        wc[e][ct][k] = M::term(w);
                        w -= M::wide_term(wc[e][ct][k]);
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kK; ++k)
                if (there(k)) {
#pragma unroll
                    for (int rt = 2 * k; rt < 2 * k + 2; ++rt) {
                        const Pair b = M::pair(M::template b_column<kDA>(lb, sb, rt, lane),
                                               M::template b_column<kDA>(lb, sb + 1, rt, lane));
#pragma unroll
                        for (int ct = 0; ct < kCT; ++ct)
                            X[rt][ct] = M::mma_terms(X[rt][ct], b, wc[0][ct], wc[1][ct]);
                    }
                }
        }
    }
    if constexpr (kStates) {
        float* w = S.states + (static_cast<long long>(bh) * nseg + seg) * state_size;
        each_place([&](float x, int at) { return w[at] = x; });
    } else {
        // steps past the sequence's end
        for (int i = max(begin, len) + wave; i < end; i += kW) {
            const long long at = batch * S.y_stride[0] + i * S.y_stride[1] + h * S.y_stride[2];
            for (int col = col0 + lane; col < col0 + dc_here; col += 64)
                if (S.y_f32) static_cast<float*>(S.y)[at + col] = 0.f;
                else static_cast<typename In::Elem*>(S.y)[at + col] = static_cast<typename In::Elem>(0.f);
        }
        if (S.state_out && seg == A.nseg - 1) {
            float* w = S.state_out + bh * state_size;
            each_place([&](float x, int at) { return w[at] = x; });
        }
    }
}

// Segments' own states to the states that enter the segments after them, in place; kV values
// a thread.
template <int kV>
__global__ void __launch_bounds__(kThreads) k_join(ChunkArgs A) {
    typedef float Vec __attribute__((ext_vector_type(kV)));
    const JobArgs& S = job_of(blockIdx.z);
    const int nseg = A.nseg - 1, size = S.da * S.dc / kV;
    const int bh = blockIdx.y, e = blockIdx.x * kThreads + threadIdx.x;
    if (e >= size) return;
    const int batch = bh / S.heads, h = bh - batch * S.heads;
    const int len = S.lengths ? min(max(S.lengths[batch], 0), S.time) : S.time;
    const float g = decay_of(S.log_decay[h]);
    Vec* w = reinterpret_cast<Vec*>(S.states) + static_cast<long long>(bh) * nseg * size + e;
    // the segments' loads do not wait for each other
    constexpr int kAhead = 16;
    Vec x = {}, next[kAhead];
    for (int s0 = 0; s0 < nseg; s0 += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (s0 + k < nseg) next[k] = w[static_cast<long long>(s0 + k) * size];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int s = s0 + k;
            if (s < nseg) {
                const int n = min(max(len - s * A.seg_steps, 0), A.seg_steps);
                x = x * expf(g * static_cast<float>(n)) + next[k];
                w[static_cast<long long>(s) * size] = x;
            }
        }
    }
}

// Adds up what the heads that share an input hold, in head order: part is (n, heads, d) fp32,
// out (n, kept, d).
template <class T>
__global__ void k_share(const float* part, T* out, long long n, int heads, int kept, int d) {
    const int each = heads / kept;
    for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < n * kept * d;
         e += static_cast<long long>(gridDim.x) * blockDim.x) {
        const long long rest = e / d;
        const int i = static_cast<int>(e - rest * d);
        const float* p = part + rest * each * d + i;
        float sum = 0.f;
        for (int k = 0; k < each; ++k) sum += p[static_cast<long long>(k) * d];
        out[e] = from_f32<T>(sum);
    }
}

hipStream_t stream_of(const hx_attention_args& A) { return static_cast<hipStream_t>(A.stream); }

struct Operand {
    const void* p;
    const int64_t* stride;
    int64_t heads, d;
};

// How a sum is cut: state rows padded, waves and their 16-column tiles.
struct Cut {
    int rows, waves, tiles;
    int width() const { return waves * tiles * 16; }
};

Cut cut_of(int64_t type, int64_t da, int64_t dc) {
    Cut c{};
    c.rows = da <= 32 ? 32 : da <= 64 ? 64 : da <= 128 ? 128 : 256;
    c.waves = dc <= 32 ? 2 : 4;
    c.tiles = 1;
    if (dc > 64 && c.rows < 256) {
        // 128 columns: in 16 bits two tiles a wave (LDS reads serve twice: 224 us for 65536 steps, 8
        // heads, 128 x 128 in bf16, against 295 with eight waves of one); fp32 products take so much
        // longer that more waves pay instead (777 steps, 156 sequences and heads, 96 x 80: 115 us
        // against 136)
        if (type != HX_F32) {
            c.tiles = 2;
        } else {
            c.waves = 8;
            c.rows = std::max(c.rows, 64);
        }
    }
    return c;
}

// Segments of the steps, the same for all sums of a call: 512 workgroups in all, two chunks or
// more each.  Two segments would read twice what they halve, and three of one chunk or two wait
// longer for two more launches than for the chunks: forward and backward, bf16, 4 heads of 64,
// 500 steps 46 us cut and 51 whole, but 16 sequences of 300 steps 50 cut in two and 37 whole.
struct Segments {
    int count, steps;
};

Segments segments_of(const hx_attention_args& A) {
    const int chunk = with_type(A.type, [](auto t) { return InputOf<decltype(t)>::Math::kC; });
    const int width = cut_of(A.type, A.dk, A.dv).width();
    const int64_t units = A.batch * A.heads * ((A.dv + width - 1) / width);
    const int64_t chunks = std::max<int64_t>(1, (A.time + chunk - 1) / chunk);
    const int64_t want = std::min<int64_t>(512 / std::max<int64_t>(units, 1), chunks / 2);
    const int64_t each = want < 3 ? chunks : (chunks + want - 1) / want;
    return {static_cast<int>((chunks + each - 1) / each), static_cast<int>(each * chunk)};
}

ScanArgs scan_args(const hx_attention_args& A, const Operand& a, const Operand& b, const Operand& c, bool reverse) {
    ScanArgs S{};
    S.a = a.p, S.b = b.p, S.c = c.p;
    for (int i = 0; i < 3; ++i) S.a_stride[i] = a.stride[i], S.b_stride[i] = b.stride[i], S.c_stride[i] = c.stride[i];
    S.a_each = static_cast<int>(A.heads / a.heads), S.b_each = static_cast<int>(A.heads / b.heads);
    S.c_each = static_cast<int>(A.heads / c.heads);
    S.heads = static_cast<int>(A.heads), S.da = static_cast<int>(a.d), S.dc = static_cast<int>(c.d);
    S.time = static_cast<int>(A.time);
    S.reverse = reverse, S.scale_in = reverse ? static_cast<float>(A.scale) : 1.f;
    S.scale_out = reverse ? 1.f : static_cast<float>(A.scale);
    S.log_decay = A.log_decay, S.lengths = A.lengths;
    return S;
}

// Strides of a contiguous (batch, time, heads, d) array.
void contiguous(long long* s, int64_t time, int64_t heads, int64_t d) {
    s[0] = time * heads * d, s[1] = heads * d, s[2] = d;
}

template <class T, int kDA, int kW, int kCT, bool kWhole, bool kFull>
hipError_t launch_cut(ChunkArgs& A, int jobs, bool states, long long bh, hipStream_t st) {
    A.nslice = (A.job[0].dc + kW * kCT * 16 - 1) / (kW * kCT * 16);
    A.jobs = jobs;
    const dim3 grid(static_cast<unsigned>(bh * (A.nseg - states) * A.nslice * jobs));
    if (states) k_chunk<T, kDA, kW, kCT, kWhole, kFull, true><<<grid, kW * 64, 0, st>>>(A);
    else k_chunk<T, kDA, kW, kCT, kWhole, kFull, false><<<grid, kW * 64, 0, st>>>(A);
    return hipGetLastError();
}

// The jobs of one launch are of one size.
template <class T>
hipError_t launch_chunks(ChunkArgs A, int jobs, bool states, long long bh, hipStream_t st) {
    constexpr int kP = InputOf<T>::Math::kPiece;
    constexpr long long kFar = 1 << 23;          // elements from step to step: 64 of them in 32 bits of bytes
    const Cut c = cut_of(InputOf<T>::kType, A.job[0].da, A.job[0].dc);
    bool all_whole = A.job[0].da % kP == 0 && A.job[0].dc % kP == 0;
    for (int i = 0; i < jobs; ++i) {
        const ScanArgs& S = A.job[i];
        for (long long stride : {S.a_stride[1], S.b_stride[1], S.c_stride[1], S.y_stride[1]})
            all_whole = all_whole && stride >= 0 && stride < kFar;
    }
    const bool full = A.job[0].da == c.rows && A.job[0].dc % c.width() == 0;
    auto go = [&](auto rows, auto whole, auto fills) {
        constexpr int kDA = decltype(rows)::value;
        constexpr bool kWhole = decltype(whole)::value, kFull = decltype(fills)::value;
        if (c.waves == 2) return launch_cut<T, kDA, 2, 1, kWhole, kFull>(A, jobs, states, bh, st);
        if constexpr (InputOf<T>::kType != HX_F32) {
            if constexpr (kDA < 256)
                if (c.tiles == 2) return launch_cut<T, kDA, 4, 2, kWhole, kFull>(A, jobs, states, bh, st);
        } else if constexpr (kDA == 64 || kDA == 128) {
            if (c.waves == 8) return launch_cut<T, kDA, 8, 1, kWhole, kFull>(A, jobs, states, bh, st);
        }
        return launch_cut<T, kDA, 4, 1, kWhole, kFull>(A, jobs, states, bh, st);
    };
    auto rows = [&](auto whole, auto fills) {
        switch (c.rows) {
            case 32: return go(std::integral_constant<int, 32>{}, whole, fills);
            case 64: return go(std::integral_constant<int, 64>{}, whole, fills);
            case 128: return go(std::integral_constant<int, 128>{}, whole, fills);
            default: return go(std::integral_constant<int, 256>{}, whole, fills);
        }
    };
    if (all_whole && full) return rows(std::true_type{}, std::true_type{});
    return all_whole ? rows(std::true_type{}, std::false_type{}) : rows(std::false_type{}, std::false_type{});
}

// What enters each segment but the first, where there are several; the jobs are of one size.
template <class T>
hipError_t launch_states(const ChunkArgs& A, int jobs, long long bh, hipStream_t st) {
    if (A.nseg < 2) return hipSuccess;
    const hipError_t e = launch_chunks<T>(A, jobs, true, bh, st);
    if (e != hipSuccess) return e;
    // (several segments are made of 512 sequences and heads at most: within a grid's second dimension)
    const int size = A.job[0].da * A.job[0].dc, width = size % 4 == 0 ? 4 : 1;
    const dim3 grid((size / width + kThreads - 1) / kThreads, static_cast<unsigned>(bh), jobs);
    if (width == 4) k_join<4><<<grid, kThreads, 0, st>>>(A);
    else k_join<1><<<grid, kThreads, 0, st>>>(A);
    return hipGetLastError();
}

// Workspace: the segments' states (of the gradient's two directions), then fp32 gradients by head
// for each input that heads share.
size_t state_part(const hx_attention_args& A) {
    const size_t n = sizeof(float) * (segments_of(A).count - 1) * A.batch * A.heads * A.dk * A.dv;
    return (n + 255) / 256 * 256;
}

size_t shared_part(const hx_attention_args& A, int64_t heads, int64_t d) {
    const size_t n = heads == A.heads ? 0 : sizeof(float) * A.batch * A.time * A.heads * d;
    return (n + 255) / 256 * 256;
}

}  // namespace

size_t attention_workspace(const hx_attention_args& A, bool grad) {
    if (!grad) return state_part(A);
    return 2 * state_part(A) + shared_part(A, A.q_heads, A.dk) + shared_part(A, A.k_heads, A.dk) +
           shared_part(A, A.v_heads, A.dv);
}

hipError_t attention_forward(const hx_attention_args& A) {
    const Operand q{A.q, A.q_stride, A.q_heads, A.dk}, k{A.k, A.k_stride, A.k_heads, A.dk},
        v{A.v, A.v_stride, A.v_heads, A.dv};
    const Segments seg = segments_of(A);
    ChunkArgs C{};
    C.nseg = seg.count, C.seg_steps = seg.steps;
    ScanArgs& S = C.job[0];
    S = scan_args(A, q, k, v, false);
    S.states = static_cast<float*>(A.workspace);
    S.state_in = A.initial_state, S.state_out = A.end_state, S.row_stride = S.dc, S.col_stride = 1;
    S.y = A.o;
    for (int i = 0; i < 3; ++i) S.y_stride[i] = A.o_stride[i];
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        const hipError_t e = launch_states<T>(C, 1, A.batch * A.heads, stream_of(A));
        return e != hipSuccess ? e : launch_chunks<T>(C, 1, false, A.batch * A.heads, stream_of(A));
    });
}

hipError_t attention_step(const hx_attention_args& A) {
    const Operand q{A.q, A.q_stride, A.q_heads, A.dk}, k{A.k, A.k_stride, A.k_heads, A.dk},
        v{A.v, A.v_stride, A.v_heads, A.dv};
    ScanArgs S = scan_args(A, q, k, v, false);
    S.y = A.o;
    for (int i = 0; i < 3; ++i) S.y_stride[i] = A.o_stride[i];
    // four columns a lane where every row of a state starts at a whole 16 bytes
    const bool wide = S.dc % 4 == 0 && reinterpret_cast<uintptr_t>(A.state) % 16 == 0;
    int lanes = 1;
    while (lanes * (wide ? 4 : 1) < S.dc) lanes *= 2;
    const unsigned grid = static_cast<unsigned>(A.batch * S.heads);
    return with_type(A.type, [&](auto t) {
        using T = decltype(t);
        if (wide) k_step<T, 4><<<grid, kThreads, 0, stream_of(A)>>>(S, A.state, A.slots, A.n_slots, lanes);
        else k_step<T, 1><<<grid, kThreads, 0, stream_of(A)>>>(S, A.state, A.slots, A.n_slots, lanes);
        return hipGetLastError();
    });
}

hipError_t attention_backward(const hx_attention_args& A) {
    const Operand q{A.q, A.q_stride, A.q_heads, A.dk}, k{A.k, A.k_stride, A.k_heads, A.dk},
        v{A.v, A.v_stride, A.v_heads, A.dv}, o{A.grad_o, A.grad_o_stride, A.heads, A.dv};
    const hipStream_t st = stream_of(A);
    const Segments seg = segments_of(A);
    char* const space = static_cast<char*>(A.workspace);
    float* const ahead = reinterpret_cast<float*>(space);
    float* const back = reinterpret_cast<float*>(space + state_part(A));
    char* by_head = space + 2 * state_part(A);
    const int dv = static_cast<int>(A.dv);
    const long long bh = A.batch * A.heads;

    // States lie as (dk, dv) whichever way a sum takes them: k v^T going forward, q do^T going
    // back, the latter for dk and dv alike.
    enum Columns { kOfKeys, kOfValues };
    auto sum = [&](const Operand& a, const Operand& b, const Operand& c, bool reverse, Columns columns, float* states,
                   void* y, int64_t kept) {
        ScanArgs S = scan_args(A, a, b, c, reverse);
        S.row_stride = columns == kOfKeys ? 1 : dv, S.col_stride = columns == kOfKeys ? dv : 1;
        S.states = states, S.state_in = reverse ? A.grad_end : A.initial_state;
        S.y = y, S.y_f32 = kept != A.heads;
        if (S.y_f32) {
            S.y = by_head;
            by_head += shared_part(A, kept, c.d);
        }
        contiguous(S.y_stride, A.time, A.heads, c.d);
        return S;
    };
    ChunkArgs states{}, grads{};
    states.nseg = grads.nseg = seg.count;
    states.seg_steps = grads.seg_steps = seg.steps;
    states.job[0] = sum(q, k, v, false, kOfValues, ahead, nullptr, A.heads);
    states.job[1] = sum(k, q, o, true, kOfValues, back, nullptr, A.heads);
    grads.job[0] = sum(o, v, k, false, kOfKeys, ahead, A.grad_q, A.q_heads);
    grads.job[1] = sum(v, o, q, true, kOfKeys, back, A.grad_k, A.k_heads);
    grads.job[2] = sum(k, q, o, true, kOfValues, back, A.grad_v, A.v_heads);
    grads.job[2].state_out = A.grad_initial;

    return with_type(A.type, [&](auto t) -> hipError_t {
        using T = decltype(t);
        hipError_t e = launch_states<T>(states, 2, bh, st);
        if (e != hipSuccess) return e;
        if (A.dk == A.dv) {
            e = launch_chunks<T>(grads, 3, false, bh, st);
        } else {
            ChunkArgs last = grads;
            last.job[0] = grads.job[2];
            e = launch_chunks<T>(grads, 2, false, bh, st);
            if (e == hipSuccess) e = launch_chunks<T>(last, 1, false, bh, st);
        }
        void* const outs[3] = {A.grad_q, A.grad_k, A.grad_v};
        const int64_t heads[3] = {A.q_heads, A.k_heads, A.v_heads};
        for (int i = 0; i < 3 && e == hipSuccess && A.time; ++i) {
            const ScanArgs& S = grads.job[i];
            if (!S.y_f32) continue;
            const long long n = A.batch * A.time;
            const long long blocks = std::min<long long>((n * heads[i] * S.dc + kThreads - 1) / kThreads, 1 << 16);
            k_share<T><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(
                static_cast<const float*>(S.y), static_cast<T*>(outs[i]), n, S.heads, static_cast<int>(heads[i]), S.dc);
            e = hipGetLastError();
        }
        return e;
    });
}

}  // namespace hx
