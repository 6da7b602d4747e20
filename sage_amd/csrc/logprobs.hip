// Log probabilities of given tokens, entropy and top alternatives, and their gradient, for gfx950.
// With z = scale * logits, m = max z, s = sum e^(z - m), t = sum e^(z - m) (z - m):
//   lse = m + log s;  logprob = z_token - lse;  entropy = log s - t / s;  log p_j = (z_j - m) - log s.
// Bound by memory: the logits are what is read.
#include "rows.h"

namespace {

constexpr int TOP_MAX = 64;

struct LogpP {
    const float *logits;
    const uint32_t *tokens;
    float *logprob, *entropy, *lse, *top_logprobs;
    uint32_t *top_ids;
    sg_rows rows, token_rows;
    uint32_t R, C, k;
    float scale;
};

// Rising order of the numbers, NaN below all of them, -0 equal to 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ unsigned long long top_key(float x, uint32_t j) { return ((unsigned long long)order_bits(x) << 32) | (uint32_t)~j; }

__global__ void __launch_bounds__(256) logprobs_kernel(const LogpP p) {
    __shared__ float red[256];
    __shared__ unsigned long long best[256];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float *x = p.logits + sg_row_offset(p.rows, row);
    const float inf = __builtin_inff();
    auto sum = [&](float v) {
        __syncthreads();
        red[tid] = v;
        __syncthreads();
        for (int o = 128; o > 0; o >>= 1) {
            if ((int)tid < o) red[tid] += red[tid + o];
            __syncthreads();
        }
        return red[0];
    };
    float m = -inf;
    for (uint32_t j = tid; j < p.C; j += 256) m = fmaxf(m, x[j] * p.scale);
    __syncthreads();
    red[tid] = m;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)tid < o) red[tid] = fmaxf(red[tid], red[tid + o]);
        __syncthreads();
    }
    m = red[0];
    const float shift = m == -inf ? 0.0f : m;
    float s = 0.0f, t = 0.0f;
    for (uint32_t j = tid; j < p.C; j += 256) {
        const float d = x[j] * p.scale - shift;
        const float e = expf(d);
        s += e;
        if (d != -inf) t += e * d;
    }
    s = sum(s);
    t = sum(t);
    const float logs = logf(s);
    const bool empty = m == -inf && s == 0.0f;
    if (tid == 0) {
        p.lse[row] = empty ? -inf : shift + logs;
        if (p.entropy) p.entropy[row] = empty ? 0.0f : logs - t / s;
        if (p.logprob) {
            const uint32_t tok = p.tokens[sg_row_offset(p.token_rows, row)];
            float v = 0.0f;
            if (tok < p.C) v = empty ? -inf : (x[tok] * p.scale - shift) - logs;
            p.logprob[row] = v;
        }
    }
    unsigned long long last = ~0ull;
    for (uint32_t i = 0; i < p.k; ++i) {
        unsigned long long b = 0;
        for (uint32_t j = tid; j < p.C; j += 256) {
            const unsigned long long key = top_key(x[j], j);
            if (key < last && key > b) b = key;
        }
        __syncthreads();
        best[tid] = b;
        __syncthreads();
        for (int o = 128; o > 0; o >>= 1) {
            if ((int)tid < o && best[tid + o] > best[tid]) best[tid] = best[tid + o];
            __syncthreads();
        }
        last = best[0];
        if (tid == 0) {
            const uint32_t j = ~(uint32_t)last;
            p.top_ids[(uint64_t)row * p.k + i] = j;
            p.top_logprobs[(uint64_t)row * p.k + i] = empty ? -inf : (x[j] * p.scale - shift) - logs;
        }
    }
}

struct LogpGradP {
    const float *logits;
    const uint32_t *tokens;
    const float *lse, *entropy, *g_logprob, *g_entropy;
    float *glogits;
    sg_rows rows, token_rows, gl_rows, ge_rows;
    uint32_t R, C;
    float scale;
};

__global__ void __launch_bounds__(256) logprobs_grad_kernel(const LogpGradP p) {
    const uint32_t row = blockIdx.x;
    const float *x = p.logits + sg_row_offset(p.rows, row);
    float *y = p.glogits + (uint64_t)row * p.C;
    const float inf = __builtin_inff();
    const float lse = p.lse[row];
    const uint32_t tok = p.g_logprob ? p.tokens[sg_row_offset(p.token_rows, row)] : ~0u;
    const float gl = tok < p.C ? p.g_logprob[sg_row_offset(p.gl_rows, row)] : 0.0f;
    const float ge = p.g_entropy ? p.g_entropy[sg_row_offset(p.ge_rows, row)] : 0.0f;
    const float h = p.g_entropy ? p.entropy[row] : 0.0f;
    for (uint32_t j = threadIdx.x; j < p.C; j += 256) {
        const float z = x[j] * p.scale;
        float g = 0.0f;
        if (z != -inf) {
            const float lp = z - lse, pr = expf(lp);
            g = -pr * (gl + ge * (lp + h));
            if (j == tok) g += gl;
        }
        y[j] = g * p.scale;
    }
}

// t's extents are the logits' leading ones (one element where there are none), with `more` axes behind them
int check_leading(sg_ctx *ctx, const sg_tensor *t, const sg_tensor *logits, int more, const char *who) {
    const int lead = logits->rank - 1;
    if (lead == 0 && more == 0) {
        if (t->rank != 1 || t->extents[0] != 1) return sg_fail(ctx, SG_ERR_SHAPE, "%s: one element expected", who);
        return SG_OK;
    }
    if (t->rank != lead + more) return sg_fail(ctx, SG_ERR_SHAPE, "%s: rank %d, expected %d", who, t->rank, lead + more);
    for (int i = 0; i < lead; ++i)
        if (t->extents[i] != logits->extents[i]) return sg_fail(ctx, SG_ERR_SHAPE, "%s: extent[%d] differs from the logits'", who, i);
    return SG_OK;
}

int check_row_output(sg_ctx *ctx, const sg_tensor *t, const sg_tensor *logits, const char *who) {
    int rc;
    if ((rc = sg_check_f32(ctx, t, who)) != SG_OK) return rc;
    if ((rc = check_leading(ctx, t, logits, 0, who)) != SG_OK) return rc;
    if (!sg_is_dense(t)) return sg_fail(ctx, SG_ERR_SHAPE, "%s: must be dense row-major", who);
    return SG_OK;
}

int check_logits(sg_ctx *ctx, const sg_tensor *logits, float scale, const char *who) {
    int rc;
    if ((rc = sg_check_f32(ctx, logits, who)) != SG_OK) return rc;
    if (logits->extents[logits->rank - 1] > 1 && logits->strides[logits->rank - 1] != 1)
        return sg_fail(ctx, SG_ERR_SHAPE, "%s: the last axis must have unit stride", who);
    if (!(scale > 0.0f) || scale > 3.4028234e38f) return sg_fail(ctx, SG_ERR_ARG, "%s: scale must be positive and finite", who);
    return SG_OK;
}

int check_tokens(sg_ctx *ctx, const sg_tensor *tokens, const sg_tensor *logits, const char *who) {
    int rc;
    if ((rc = sg_check_index(ctx, tokens, who)) != SG_OK) return rc;
    return check_leading(ctx, tokens, logits, 0, who);
}

float *f32_ptr(const sg_tensor *t) { return t ? (float *)t->base + t->offset : nullptr; }

}  // namespace

extern "C" int sg_token_logprobs(sg_ctx *ctx, const sg_tensor *logits, const sg_tensor *tokens, float scale, const sg_tensor *logprob,
                                 const sg_tensor *entropy, const sg_tensor *lse, const sg_tensor *top_ids, const sg_tensor *top_logprobs) {
    int rc;
    if ((rc = check_logits(ctx, logits, scale, "sg_token_logprobs logits")) != SG_OK) return rc;
    if (tokens && (rc = check_tokens(ctx, tokens, logits, "sg_token_logprobs tokens")) != SG_OK) return rc;
    if (logprob && !tokens) return sg_fail(ctx, SG_ERR_ARG, "sg_token_logprobs: logprob needs tokens");
    if (logprob && (rc = check_row_output(ctx, logprob, logits, "sg_token_logprobs logprob")) != SG_OK) return rc;
    if (entropy && (rc = check_row_output(ctx, entropy, logits, "sg_token_logprobs entropy")) != SG_OK) return rc;
    if ((rc = check_row_output(ctx, lse, logits, "sg_token_logprobs lse")) != SG_OK) return rc;
    if (!top_ids != !top_logprobs) return sg_fail(ctx, SG_ERR_ARG, "sg_token_logprobs: top_ids and top_logprobs come together");
    const int lead = logits->rank - 1;
    const int64_t C = logits->extents[lead];
    int64_t k = 0;
    if (top_ids) {
        if ((rc = sg_validate_tensor(ctx, top_ids, "sg_token_logprobs top_ids")) != SG_OK) return rc;
        if ((rc = sg_check_f32(ctx, top_logprobs, "sg_token_logprobs top_logprobs")) != SG_OK) return rc;
        if (top_ids->dtype != SG_UINT) return sg_fail(ctx, SG_ERR_DTYPE, "sg_token_logprobs top_ids: uint expected");
        if ((rc = check_leading(ctx, top_ids, logits, 1, "sg_token_logprobs top_ids")) != SG_OK) return rc;
        if ((rc = check_leading(ctx, top_logprobs, logits, 1, "sg_token_logprobs top_logprobs")) != SG_OK) return rc;
        k = top_ids->extents[lead];
        if (top_logprobs->extents[lead] != k) return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs: top_ids and top_logprobs differ in size");
        if (k > TOP_MAX || k > C) return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs: %lld alternatives of %lld (at most %d)", (long long)k, (long long)C, TOP_MAX);
        if (!sg_is_dense(top_ids) || !sg_is_dense(top_logprobs)) return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs: top_ids and top_logprobs must be dense row-major");
    }
    if (!ctx) return SG_ERR_ARG;
    LogpP p{};
    p.logits = f32_ptr(logits);
    p.R = (uint32_t)sg_make_rows(logits, lead, &p.rows);
    if (tokens) {
        p.tokens = (const uint32_t *)tokens->base + tokens->offset;
        (void)sg_make_rows(tokens, tokens->rank, &p.token_rows);
    }
    p.logprob = f32_ptr(logprob);
    p.entropy = f32_ptr(entropy);
    p.lse = f32_ptr(lse);
    p.top_ids = top_ids ? (uint32_t *)top_ids->base + top_ids->offset : nullptr;
    p.top_logprobs = f32_ptr(top_logprobs);
    p.C = (uint32_t)C;
    p.k = (uint32_t)k;
    p.scale = scale;
    sg_device_guard guard(ctx);
    hipLaunchKernelGGL(logprobs_kernel, dim3(p.R), dim3(256), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "token_logprobs");
    return SG_OK;
}

extern "C" int sg_token_logprobs_grad(sg_ctx *ctx, const sg_tensor *logits, const sg_tensor *tokens, float scale, const sg_tensor *lse,
                                      const sg_tensor *entropy, const sg_tensor *g_logprob, const sg_tensor *g_entropy, const sg_tensor *glogits) {
    int rc;
    if ((rc = check_logits(ctx, logits, scale, "sg_token_logprobs_grad logits")) != SG_OK) return rc;
    if (tokens && (rc = check_tokens(ctx, tokens, logits, "sg_token_logprobs_grad tokens")) != SG_OK) return rc;
    if ((rc = check_row_output(ctx, lse, logits, "sg_token_logprobs_grad lse")) != SG_OK) return rc;
    if (entropy && (rc = check_row_output(ctx, entropy, logits, "sg_token_logprobs_grad entropy")) != SG_OK) return rc;
    if (!g_logprob && !g_entropy) return sg_fail(ctx, SG_ERR_ARG, "sg_token_logprobs_grad: no gradient given");
    if (g_logprob && !tokens) return sg_fail(ctx, SG_ERR_ARG, "sg_token_logprobs_grad: g_logprob needs tokens");
    if (g_entropy && !entropy) return sg_fail(ctx, SG_ERR_ARG, "sg_token_logprobs_grad: g_entropy needs entropy");
    if (g_logprob && (rc = sg_check_f32(ctx, g_logprob, "sg_token_logprobs_grad g_logprob")) != SG_OK) return rc;
    if (g_logprob && (rc = check_leading(ctx, g_logprob, logits, 0, "sg_token_logprobs_grad g_logprob")) != SG_OK) return rc;
    if (g_entropy && (rc = sg_check_f32(ctx, g_entropy, "sg_token_logprobs_grad g_entropy")) != SG_OK) return rc;
    if (g_entropy && (rc = check_leading(ctx, g_entropy, logits, 0, "sg_token_logprobs_grad g_entropy")) != SG_OK) return rc;
    if ((rc = sg_check_f32(ctx, glogits, "sg_token_logprobs_grad glogits")) != SG_OK) return rc;
    if (glogits->rank != logits->rank) return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs_grad: glogits' rank differs from the logits'");
    for (int i = 0; i < logits->rank; ++i)
        if (glogits->extents[i] != logits->extents[i]) return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs_grad: glogits' extent[%d] differs from the logits'", i);
    if (!sg_is_dense(glogits)) return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs_grad: glogits must be dense row-major");
    if (!ctx) return SG_ERR_ARG;
    const int lead = logits->rank - 1;
    LogpGradP p{};
    p.logits = f32_ptr(logits);
    p.R = (uint32_t)sg_make_rows(logits, lead, &p.rows);
    if (g_logprob) {
        p.tokens = (const uint32_t *)tokens->base + tokens->offset;
        (void)sg_make_rows(tokens, tokens->rank, &p.token_rows);
        p.g_logprob = f32_ptr(g_logprob);
        (void)sg_make_rows(g_logprob, g_logprob->rank, &p.gl_rows);
    }
    if (g_entropy) {
        p.entropy = f32_ptr(entropy);
        p.g_entropy = f32_ptr(g_entropy);
        (void)sg_make_rows(g_entropy, g_entropy->rank, &p.ge_rows);
    }
    p.lse = f32_ptr(lse);
    p.glogits = f32_ptr(glogits);
    p.C = (uint32_t)logits->extents[lead];
    p.scale = scale;
    sg_device_guard guard(ctx);
    hipLaunchKernelGGL(logprobs_grad_kernel, dim3(p.R), dim3(256), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "token_logprobs_grad");
    return SG_OK;
}
