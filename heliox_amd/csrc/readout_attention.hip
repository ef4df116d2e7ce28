// Linear attention with a decay for each head.  Outputs and gradients are the same sum over
// different operands,
//
//   y_i = sum over j <= i of e^{g (i - j)} (a_i . b_j) c_j + (what a state brings in),
//
// with i counting steps from the sequence's first (forward) or last (reverse):
//   o:  a, b, c = q, k, v   forward, state k v^T        dq: a, b, c = do, v, k  forward, state v k^T
//   dk: a, b, c = v, do, q  reverse, state do q^T       dv: a, b, c = k, q, do  reverse, state q do^T
#include <algorithm>

#include "readout.h"

namespace hx {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 16;                     // state columns of one workgroup
constexpr int kParts = kThreads / kCols;      // lanes that share a column's rows

struct ScanArgs {
    const void *a, *b, *c;
    long long a_stride[3], b_stride[3], c_stride[3];
    int a_heads, b_heads, c_heads, heads, da, dc, time, ncol;
    bool reverse;
    float scale_in, scale_out;       // of what enters the state, and of y
    const float* log_decay;
    const int32_t* lengths;
    const float* state_in;
    float* state_out;
    int row_stride, col_stride;      // of a state's da and dc
    const int32_t* slots;            // states by slot instead of by sequence
    long long n_slots;
    bool by_slot;
    void* y;
    long long y_stride[3];
    int y_heads;
};

// One workgroup per (sequence, head, 16 state columns), one step after another: a column's
// rows lie over 16 lanes, so that y is one shuffled sum.
template <class T, class Y>
__global__ void __launch_bounds__(kThreads) k_scan(ScanArgs S) {
    const int col = blockIdx.x % S.ncol * kCols + threadIdx.x / kParts;
    const int bh = blockIdx.x / S.ncol;
    const int batch = bh / S.heads, h = bh - batch * S.heads;
    const int part = threadIdx.x % kParts;
    const bool mine = col < S.dc;
    const int len = S.lengths ? min(max(S.lengths[batch], 0), S.time) : S.time;
    const float decay = expf(S.log_decay[h]);
    long long slot = batch;
    if (S.by_slot && S.slots) slot = S.slots[batch];
    const bool run = !S.by_slot || (slot >= 0 && slot < S.n_slots);
    const long long at = (slot * S.heads + h) * static_cast<long long>(S.da) * S.dc +
                         static_cast<long long>(col) * S.col_stride;
    const T* a = static_cast<const T*>(S.a) + batch * S.a_stride[0] + (h * S.a_heads / S.heads) * S.a_stride[2];
    const T* b = static_cast<const T*>(S.b) + batch * S.b_stride[0] + (h * S.b_heads / S.heads) * S.b_stride[2];
    const T* c = static_cast<const T*>(S.c) + batch * S.c_stride[0] + (h * S.c_heads / S.heads) * S.c_stride[2];
    Y* y = static_cast<Y*>(S.y) + batch * S.y_stride[0] + h * S.y_stride[2];
    float s[kAttnMaxDim / kParts];
#pragma unroll
    for (int i = 0; i < kAttnMaxDim / kParts; ++i) {
        const int row = i * kParts + part;
        s[i] = run && mine && row < S.da && S.state_in ? S.state_in[at + static_cast<long long>(row) * S.row_stride] : 0.f;
    }
    for (int i = 0; i < S.time; ++i) {
        const int t = S.reverse && i < len ? len - 1 - i : i;
        float sum = 0.f;
        if (run && i < len && mine) {
            const float ct = to_f32(c[t * S.c_stride[1] + col]) * S.scale_in;
            // a state that enters in reverse has not decayed before the last step
            const float keep = S.reverse && i == 0 ? 1.f : decay;
#pragma unroll
            for (int r = 0; r < kAttnMaxDim / kParts; ++r) {
                const int row = r * kParts + part;
                if (row < S.da) {
                    s[r] = fmaf(to_f32(b[t * S.b_stride[1] + row]), ct, s[r] * keep);
                    sum = fmaf(to_f32(a[t * S.a_stride[1] + row]), s[r], sum);
                }
            }
        }
        for (int m = kParts / 2; m > 0; m >>= 1) sum += __shfl_xor(sum, m);
        if (mine && part == 0) y[t * S.y_stride[1] + col] = from_f32<Y>(sum * S.scale_out);
    }
    if (S.state_out && run && mine) {
        const float keep = S.reverse && len ? decay : 1.f;
#pragma unroll
        for (int r = 0; r < kAttnMaxDim / kParts; ++r) {
            const int row = r * kParts + part;
            if (row < S.da) S.state_out[at + static_cast<long long>(row) * S.row_stride] = s[r] * keep;
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

template <class T, class Y>
hipError_t launch_scan(const ScanArgs& S, long long batch, hipStream_t st) {
    k_scan<T, Y><<<static_cast<unsigned>(batch * S.heads * S.ncol), kThreads, 0, st>>>(S);
    return hipGetLastError();
}

struct Operand {
    const void* p;
    const int64_t* stride;
    int64_t heads, d;
};

ScanArgs scan_args(const hx_attention_args& A, const Operand& a, const Operand& b, const Operand& c, bool reverse) {
    ScanArgs S{};
    S.a = a.p, S.b = b.p, S.c = c.p;
    for (int i = 0; i < 3; ++i) S.a_stride[i] = a.stride[i], S.b_stride[i] = b.stride[i], S.c_stride[i] = c.stride[i];
    S.a_heads = static_cast<int>(a.heads), S.b_heads = static_cast<int>(b.heads), S.c_heads = static_cast<int>(c.heads);
    S.heads = static_cast<int>(A.heads), S.da = static_cast<int>(a.d), S.dc = static_cast<int>(c.d);
    S.time = static_cast<int>(A.time), S.ncol = (S.dc + kCols - 1) / kCols;
    S.reverse = reverse, S.scale_in = reverse ? static_cast<float>(A.scale) : 1.f;
    S.scale_out = reverse ? 1.f : static_cast<float>(A.scale);
    S.log_decay = A.log_decay, S.lengths = A.lengths;
    return S;
}

// Strides of a contiguous (batch, time, heads, d) array.
void contiguous(long long* s, int64_t time, int64_t heads, int64_t d) {
    s[0] = time * heads * d, s[1] = heads * d, s[2] = d;
}

size_t shared_part(const hx_attention_args& A, int64_t heads, int64_t d) {
    return heads == A.heads ? 0 : sizeof(float) * A.batch * A.time * A.heads * d;
}

}  // namespace

size_t attention_workspace(const hx_attention_args& A, bool grad) {
    if (!grad) return 0;
    return std::max({shared_part(A, A.q_heads, A.dk), shared_part(A, A.k_heads, A.dk), shared_part(A, A.v_heads, A.dv)});
}

hipError_t attention_forward(const hx_attention_args& A) {
    const Operand q{A.q, A.q_stride, A.q_heads, A.dk}, k{A.k, A.k_stride, A.k_heads, A.dk},
        v{A.v, A.v_stride, A.v_heads, A.dv};
    ScanArgs S = scan_args(A, q, k, v, false);
    S.state_in = A.initial_state, S.state_out = A.end_state, S.row_stride = S.dc, S.col_stride = 1;
    S.y = A.o;
    for (int i = 0; i < 3; ++i) S.y_stride[i] = A.o_stride[i];
    return with_type(A.type, [&](auto t) { return launch_scan<decltype(t), decltype(t)>(S, A.batch, stream_of(A)); });
}

hipError_t attention_step(const hx_attention_args& A) {
    const Operand q{A.q, A.q_stride, A.q_heads, A.dk}, k{A.k, A.k_stride, A.k_heads, A.dk},
        v{A.v, A.v_stride, A.v_heads, A.dv};
    ScanArgs S = scan_args(A, q, k, v, false);
    S.lengths = nullptr;
    S.state_in = S.state_out = A.state, S.row_stride = S.dc, S.col_stride = 1;
    S.by_slot = true, S.slots = A.slots, S.n_slots = A.n_slots;
    S.y = A.o;
    for (int i = 0; i < 3; ++i) S.y_stride[i] = A.o_stride[i];
    return with_type(A.type, [&](auto t) { return launch_scan<decltype(t), decltype(t)>(S, A.batch, stream_of(A)); });
}

hipError_t attention_backward(const hx_attention_args& A) {
    const Operand q{A.q, A.q_stride, A.q_heads, A.dk}, k{A.k, A.k_stride, A.k_heads, A.dk},
        v{A.v, A.v_stride, A.v_heads, A.dv}, o{A.grad_o, A.grad_o_stride, A.heads, A.dv};
    const hipStream_t st = stream_of(A);
    auto one = [&](const Operand& a, const Operand& b, const Operand& c, bool reverse, bool transposed,
                   const float* in, float* out, void* y, int64_t kept) -> hipError_t {
        ScanArgs S = scan_args(A, a, b, c, reverse);
        S.state_in = in, S.state_out = out;
        S.row_stride = transposed ? 1 : S.dc, S.col_stride = transposed ? S.da : 1;
        const bool shared = kept != A.heads;
        S.y = shared ? A.workspace : y;
        contiguous(S.y_stride, A.time, A.heads, c.d);
        return with_type(A.type, [&](auto t) -> hipError_t {
            using T = decltype(t);
            if (!shared) return launch_scan<T, T>(S, A.batch, st);
            hipError_t e = launch_scan<T, float>(S, A.batch, st);
            if (e != hipSuccess || !A.time) return e;
            const long long n = A.batch * A.time;
            const long long blocks = std::min<long long>((n * kept * c.d + kThreads - 1) / kThreads, 1 << 16);
            k_share<T><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(
                static_cast<const float*>(A.workspace), static_cast<T*>(y), n, S.heads, static_cast<int>(kept),
                static_cast<int>(c.d));
            return hipGetLastError();
        });
    };
    hipError_t e = one(o, v, k, false, true, A.initial_state, nullptr, A.grad_q, A.q_heads);
    if (e == hipSuccess) e = one(v, o, q, true, true, A.grad_end, nullptr, A.grad_k, A.k_heads);
    if (e == hipSuccess) e = one(k, q, o, true, false, A.grad_end, A.grad_initial, A.grad_v, A.v_heads);
    return e;
}

}  // namespace hx
