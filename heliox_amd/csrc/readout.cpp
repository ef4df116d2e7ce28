// C entry points of the readout operators: argument checks, empty problems, error texts.
#include "readout.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace {

thread_local char g_error[512];

int refuse(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof g_error, fmt, ap);
    va_end(ap);
    return -1;
}

int launched(const char* call, hipError_t e) {
    return e == hipSuccess ? 0 : refuse("%s: %s", call, hipGetErrorString(e));
}

bool known_type(int64_t t) { return t == HX_F32 || t == HX_F16 || t == HX_BF16; }

constexpr int64_t kMaxRows = 1 << 21;     // of 1024 threads each: a grid has under 2^32

int64_t checked_product(int64_t a, int64_t b) {
    int64_t p = 0;
    return __builtin_mul_overflow(a, b, &p) ? INT64_MAX : p;
}

// Sizes shared by the attention's calls; a text's call name comes first.
int attention_sizes(const char* call, const hx_attention_args* A) {
    if (!A) return refuse("%s: no arguments", call);
    if (!known_type(A->type)) return refuse("%s: type %lld is not known", call, (long long)A->type);
    if (A->batch < 0 || A->time < 0) return refuse("%s: negative batch or time", call);
    if (A->heads < 1) return refuse("%s: heads has to be at least 1", call);
    const int64_t parts[3] = {A->q_heads, A->k_heads, A->v_heads};
    for (int64_t n : parts)
        if (n < 1 || A->heads % n)
            return refuse("%s: heads (%lld) is not a multiple of q_heads, k_heads and v_heads (%lld, %lld, %lld)", call,
                          (long long)A->heads, (long long)A->q_heads, (long long)A->k_heads, (long long)A->v_heads);
    if (A->dk < 1 || A->dk > hx::kAttnMaxDim || A->dv < 1 || A->dv > hx::kAttnMaxDim)
        return refuse("%s: dk (%lld) and dv (%lld) have to be in 1..%d", call, (long long)A->dk, (long long)A->dv,
                      hx::kAttnMaxDim);
    // up to twelve workgroups of 256 threads for each (sequence, head): a grid has under 2^32 threads
    if (checked_product(A->batch, A->heads) > (1 << 20) || A->time > (int64_t(1) << 30))
        return refuse("%s: batch x heads is at most 2^20 and time at most 2^30", call);
    if (!std::isfinite(A->scale)) return refuse("%s: scale is not finite", call);
    return 0;
}

int attention_inputs(const char* call, const hx_attention_args* A) {
    if (!A->q || !A->k || !A->v || !A->log_decay) return refuse("%s: q, k, v or log_decay is missing", call);
    return 0;
}

// The states that a call writes are not those it reads: workgroups of other segments read them
// while the last one writes.
int attention_states(const char* call, const hx_attention_args* A, const float* out, const char* out_name, const float* in,
                     const char* in_name) {
    const uintptr_t bytes = sizeof(float) * A->batch * A->heads * A->dk * A->dv;
    const uintptr_t o = reinterpret_cast<uintptr_t>(out), i = reinterpret_cast<uintptr_t>(in);
    if (o && i && o < i + bytes && i < o + bytes) return refuse("%s: %s overlaps %s", call, out_name, in_name);
    return 0;
}

int attention_space(const char* call, const hx_attention_args* A, bool grad) {
    const size_t need = hx::attention_workspace(*A, grad);
    if (need && (!A->workspace || A->workspace_bytes < 0 || static_cast<size_t>(A->workspace_bytes) < need))
        return refuse("%s: the workspace has to hold %zu bytes", call, need);
    if (need && reinterpret_cast<uintptr_t>(A->workspace) % 16)
        return refuse("%s: the workspace has to start at a multiple of 16 bytes", call);
    return 0;
}

// grad is the logits themselves, row for row, or apart from them; its rows are apart from each other.
int distill_gradient(const char* call, const hx_distill_args* A) {
    typedef __int128 Wide;
    const int64_t size = A->type == HX_F32 ? 4 : 2;
    const Wide width = static_cast<Wide>(A->vocab) * size, gs = static_cast<Wide>(A->grad_stride) * size,
               xs = static_cast<Wide>(A->logits_stride) * size;
    if (A->rows > 1 && (gs < 0 ? -gs : gs) < width) return refuse("%s: rows of grad overlap each other", call);
    const Wide g = reinterpret_cast<uintptr_t>(A->grad), x = reinterpret_cast<uintptr_t>(A->logits);
    if (g == x && (A->rows == 1 || gs == xs)) return 0;
    auto lowest = [&](Wide at, Wide stride) { return stride < 0 ? at + (A->rows - 1) * stride : at; };
    auto end = [&](Wide at, Wide stride) { return (stride < 0 ? at : at + (A->rows - 1) * stride) + width; };
    if (end(g, gs) <= lowest(x, xs) || end(x, xs) <= lowest(g, gs)) return 0;
    // views side by side of one wider array
    const Wide step = gs < 0 ? -gs : gs, apart = step ? ((g - x) % step + step) % step : 0;
    if (A->rows > 1 && gs == xs && apart >= width && apart <= step - width) return 0;
    return refuse("%s: grad overlaps logits without being them", call);
}

}  // namespace

extern "C" {

const char* hx_readout_error(void) { return g_error; }

int64_t hx_linear_attention_workspace(const hx_attention_args* A, int grad) {
    if (attention_sizes("hx_linear_attention_workspace", A)) return -1;
    if (!A->batch) return 0;
    return static_cast<int64_t>(hx::attention_workspace(*A, grad != 0));
}

int hx_linear_attention(const hx_attention_args* A) {
    const char* call = "hx_linear_attention";
    if (attention_sizes(call, A)) return -1;
    if (!A->batch) return 0;
    if (!A->log_decay) return refuse("%s: log_decay is missing", call);
    if (A->time && attention_inputs(call, A)) return -1;
    if (A->time && !A->o) return refuse("%s: o is missing", call);
    if (attention_states(call, A, A->end_state, "end_state", A->initial_state, "initial_state")) return -1;
    if (attention_space(call, A, false)) return -1;
    return launched(call, hx::attention_forward(*A));
}

int hx_linear_attention_grad(const hx_attention_args* A) {
    const char* call = "hx_linear_attention_grad";
    if (attention_sizes(call, A)) return -1;
    if (!A->batch) return 0;
    if (!A->log_decay) return refuse("%s: log_decay is missing", call);
    if (A->time && attention_inputs(call, A)) return -1;
    if (A->time && (!A->grad_o || !A->grad_q || !A->grad_k || !A->grad_v))
        return refuse("%s: grad_o, grad_q, grad_k or grad_v is missing", call);
    if (attention_states(call, A, A->grad_initial, "grad_initial", A->initial_state, "initial_state") ||
        attention_states(call, A, A->grad_initial, "grad_initial", A->grad_end, "grad_end"))
        return -1;
    if (attention_space(call, A, true)) return -1;
    return launched(call, hx::attention_backward(*A));
}

int hx_linear_attention_step(const hx_attention_args* A) {
    const char* call = "hx_linear_attention_step";
    if (attention_sizes(call, A)) return -1;
    if (A->time != 1) return refuse("%s: time has to be 1", call);
    if (A->n_slots < 0) return refuse("%s: n_slots is negative", call);
    if (!A->slots && A->batch > A->n_slots) return refuse("%s: %lld rows, but only %lld states", call,
                                                          (long long)A->batch, (long long)A->n_slots);
    if (!A->batch) return 0;
    if (attention_inputs(call, A)) return -1;
    if (!A->o || (A->n_slots && !A->state)) return refuse("%s: o or state is missing", call);
    return launched(call, hx::attention_step(*A));
}

int hx_distill_loss(const hx_distill_args* A) {
    const char* call = "hx_distill_loss";
    if (!A) return refuse("%s: no arguments", call);
    if (!known_type(A->type) || !known_type(A->teacher_type)) return refuse("%s: type is not known", call);
    if (A->index_bits != 32 && A->index_bits != 64) return refuse("%s: indexes have 32 or 64 bits", call);
    if (A->rows < 0 || A->rows > kMaxRows) return refuse("%s: rows has to be in 0..2^21", call);
    if (A->vocab < 1 || A->vocab > hx::kDistillMaxVocab)
        return refuse("%s: vocab (%lld) has to be in 1..%lld", call, (long long)A->vocab,
                      (long long)hx::kDistillMaxVocab);
    if (A->top < 0 || A->top > hx::kDistillMaxTop)
        return refuse("%s: top (%lld) has to be in 0..%lld", call, (long long)A->top, (long long)hx::kDistillMaxTop);
    // it and its reciprocal times log2 e are fp32 numbers in the kernel
    if (!(A->temperature >= 0x1p-126) || !(A->temperature <= 0x1p126))
        return refuse("%s: temperature has to be positive, in 2^-126..2^126", call);
    if (!A->rows) return 0;
    if (!A->logits || !A->loss || (A->top && (!A->index || !A->teacher)))
        return refuse("%s: logits, index, teacher or loss is missing", call);
    if (A->grad && distill_gradient(call, A)) return -1;
    return launched(call, hx::distill_launch(*A));
}

int hx_sample(const hx_sample_args* A) {
    const char* call = "hx_sample";
    if (!A) return refuse("%s: no arguments", call);
    if (!known_type(A->type)) return refuse("%s: type is not known", call);
    if (A->rows < 0 || A->rows > kMaxRows) return refuse("%s: rows has to be in 0..2^21", call);
    // masses count to 2^40 each: 2^22 of them stay inside 63 bits
    if (A->vocab < 1 || A->vocab > (1 << 22)) return refuse("%s: vocab has to be in 1..2^22", call);
    if (!A->rows) return 0;
    if (!A->logits || !A->u || !A->token || !A->logprob)
        return refuse("%s: logits, u, token or logprob is missing", call);
    return launched(call, hx::sample_launch(*A));
}

}  // extern "C"
