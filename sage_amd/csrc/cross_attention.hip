// Cross attention of queries to the states of another sequence, forward and backward, for gfx950.
#include "rows.h"

namespace {

struct CrossP {
    const float *q, *k, *v, *mask, *out, *gout;
    float *lse;  // also read, by the gradient
    float *o, *gq, *gk, *gv;
    int N, H, G, Lq, Lk;
    // strides over batch, head and position of: q, k, v, out, gout, gq, gk, gv
    int64_t q_b, q_h, q_l, k_b, k_h, k_l, v_b, v_h, v_l, o_b, o_h, o_l, go_b, go_h, go_l, gq_b, gq_h, gq_l, gk_b, gk_h, gk_l, gv_b, gv_h, gv_l;
    int64_t mask_b;
    float scale;
};

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// A wavefront per query row, 64 keys at a time: a key per lane for the scores, a head index per lane for the sums.
template <int D>
__global__ void __launch_bounds__(64) cross_forward_kernel(const CrossP p) {
    const int lane = threadIdx.x;
    const unsigned id = blockIdx.x;
    const int l = id % p.Lq, h = id / p.Lq % p.H, b = id / p.Lq / p.H, g = h / (p.H / p.G);
    const float *q = p.q + b * p.q_b + h * p.q_h + l * p.q_l, *K = p.k + b * p.k_b + g * p.k_h, *V = p.v + b * p.v_b + g * p.v_h;
    const float inf = __builtin_inff();
    float m = -inf, s = 0.0f, acc = 0.0f;
    for (int j0 = 0; j0 < p.Lk; j0 += 64) {
        const int j = j0 + lane;
        const bool seen = j < p.Lk && (!p.mask || p.mask[b * p.mask_b + j] != 0.0f);
        float x = -inf;
        if (seen) {
            x = 0.0f;
            for (int d = 0; d < D; ++d) x += q[d] * K[j * p.k_l + d];
            x *= p.scale;
        }
        const float mn = fmaxf(m, wave_max(x));
        if (mn == -inf) continue;
        const float c = expf(m - mn), e = expf(x - mn);
        s = s * c + wave_sum(e);
        acc *= c;
        m = mn;
        for (int r = 0; r < 64; ++r) {
            const float er = __shfl(e, r, 64);
            if (__shfl((int)seen, r, 64) && lane < D) acc += er * V[(j0 + r) * p.v_l + lane];
        }
    }
    if (lane < D) p.o[b * p.o_b + h * p.o_h + l * p.o_l + lane] = s > 0.0f ? acc / s : s == s ? 0.0f : s;
    if (p.lse && lane == 0) p.lse[id] = s == 0.0f ? -inf : m + logf(s);
}

template <int D>
__global__ void __launch_bounds__(64) cross_gq_kernel(const CrossP p) {
    const int lane = threadIdx.x;
    const unsigned id = blockIdx.x;
    const int l = id % p.Lq, h = id / p.Lq % p.H, b = id / p.Lq / p.H, g = h / (p.H / p.G);
    const float *q = p.q + b * p.q_b + h * p.q_h + l * p.q_l, *K = p.k + b * p.k_b + g * p.k_h, *V = p.v + b * p.v_b + g * p.v_h;
    const float *go = p.gout + b * p.go_b + h * p.go_h + l * p.go_l, *o = p.out + b * p.o_b + h * p.o_h + l * p.o_l;
    const float lse = p.lse[id];
    const float delta = wave_sum(lane < D ? go[lane] * o[lane] : 0.0f);
    float acc = 0.0f;
    for (int j0 = 0; j0 < p.Lk; j0 += 64) {
        const int j = j0 + lane;
        const bool seen = j < p.Lk && (!p.mask || p.mask[b * p.mask_b + j] != 0.0f);
        float ds = 0.0f;
        if (seen) {
            float x = 0.0f, dp = 0.0f;
            for (int d = 0; d < D; ++d) {
                x += q[d] * K[j * p.k_l + d];
                dp += go[d] * V[j * p.v_l + d];
            }
            ds = expf(x * p.scale - lse) * (dp - delta) * p.scale;
        }
        for (int r = 0; r < 64; ++r) {
            const float dr = __shfl(ds, r, 64);
            if (__shfl((int)seen, r, 64) && lane < D) acc += dr * K[(j0 + r) * p.k_l + lane];
        }
    }
    if (lane < D) p.gq[b * p.gq_b + h * p.gq_h + l * p.gq_l + lane] = acc;
}

template <int D>
__global__ void __launch_bounds__(64) cross_gkv_kernel(const CrossP p) {
    const int lane = threadIdx.x;
    const unsigned id = blockIdx.x;
    const int j = id % p.Lk, g = id / p.Lk % p.G, b = id / p.Lk / p.G, group = p.H / p.G;
    const float *k = p.k + b * p.k_b + g * p.k_h + j * p.k_l, *v = p.v + b * p.v_b + g * p.v_h + j * p.v_l;
    float ak = 0.0f, av = 0.0f;
    if (!p.mask || p.mask[b * p.mask_b + j] != 0.0f) {
        for (int hh = 0; hh < group; ++hh) {
            const int h = g * group + hh;
            const float *Q = p.q + b * p.q_b + h * p.q_h, *GO = p.gout + b * p.go_b + h * p.go_h, *O = p.out + b * p.o_b + h * p.o_h;
            for (int l0 = 0; l0 < p.Lq; l0 += 64) {
                const int l = l0 + lane;
                float pr = 0.0f, ds = 0.0f;
                if (l < p.Lq) {
                    float x = 0.0f, dp = 0.0f, delta = 0.0f;
                    for (int d = 0; d < D; ++d) {
                        x += Q[l * p.q_l + d] * k[d];
                        dp += GO[l * p.go_l + d] * v[d];
                        delta += GO[l * p.go_l + d] * O[l * p.o_l + d];
                    }
                    pr = expf(x * p.scale - p.lse[((int64_t)b * p.H + h) * p.Lq + l]);
                    ds = pr * (dp - delta) * p.scale;
                }
                for (int r = 0; r < 64 && l0 + r < p.Lq; ++r) {
                    const float er = __shfl(pr, r, 64), dr = __shfl(ds, r, 64);
                    if (lane < D) {
                        av += er * GO[(l0 + r) * p.go_l + lane];
                        ak += dr * Q[(l0 + r) * p.q_l + lane];
                    }
                }
            }
        }
    }
    if (lane < D) {
        p.gk[b * p.gk_b + g * p.gk_h + j * p.gk_l + lane] = ak;
        p.gv[b * p.gv_b + g * p.gv_h + j * p.gv_l + lane] = av;
    }
}

int check_operand(sg_ctx *ctx, const sg_tensor *t, int64_t n, int64_t heads, int64_t len, int64_t D, const char *who, const float **ptr, int64_t *sb,
                  int64_t *sh, int64_t *sl) {
    const int rc = sg_check_f32(ctx, t, who);
    if (rc != SG_OK) return rc;
    if (t->rank != 4) return sg_fail(ctx, SG_ERR_SHAPE, "%s: rank %d, expected [batch, heads, length, head size]", who, t->rank);
    if (t->extents[0] != n || t->extents[1] != heads || t->extents[2] != len || t->extents[3] != D)
        return sg_fail(ctx, SG_ERR_SHAPE, "%s: [%lld, %lld, %lld, %lld], expected [%lld, %lld, %lld, %lld]", who, (long long)t->extents[0], (long long)t->extents[1],
                       (long long)t->extents[2], (long long)t->extents[3], (long long)n, (long long)heads, (long long)len, (long long)D);
    if (t->strides[3] != 1) return sg_fail(ctx, SG_ERR_SHAPE, "%s: the head dimension must have unit stride", who);
    *ptr = (const float *)t->base + t->offset;
    *sb = t->strides[0];
    *sh = t->strides[1];
    *sl = t->strides[2];
    return SG_OK;
}

// No two elements of an output may share an address: every axis steps over all the axes inside it.
int check_apart(sg_ctx *ctx, const sg_tensor *t, const char *who) {
    int order[4] = {0, 1, 2, 3};
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 4; ++j)
            if (t->strides[order[j]] < t->strides[order[i]]) { const int x = order[i]; order[i] = order[j]; order[j] = x; }
    int64_t reach = 0;  // the last offset inside
    for (int i = 0; i < 4; ++i) {
        const int a = order[i];
        if (t->extents[a] == 1) continue;
        if (t->strides[a] <= reach) return sg_fail(ctx, SG_ERR_SHAPE, "%s: elements share addresses", who);
        reach += (t->extents[a] - 1) * t->strides[a];
    }
    return SG_OK;
}

int check_call(sg_ctx *ctx, const sg_tensor *q, const sg_tensor *k, const sg_tensor *v, const sg_tensor *mask, const sg_tensor *out, const sg_tensor *lse,
               bool out_written, CrossP &p) {
    int rc;
    if ((rc = sg_check_f32(ctx, q, "cross attention q")) != SG_OK) return rc;
    if ((rc = sg_check_f32(ctx, k, "cross attention k")) != SG_OK) return rc;
    if (q->rank != 4 || k->rank != 4) return sg_fail(ctx, SG_ERR_SHAPE, "cross attention: q and k must be [batch, heads, length, head size]");
    const int64_t N = q->extents[0], H = q->extents[1], Lq = q->extents[2], D = q->extents[3], G = k->extents[1], Lk = k->extents[2];
    if (D != 32 && D != 64) return sg_fail(ctx, SG_ERR_SHAPE, "cross attention: head size %lld (32 and 64 are built)", (long long)D);
    if (H % G != 0) return sg_fail(ctx, SG_ERR_SHAPE, "cross attention: %lld query heads over %lld key heads", (long long)H, (long long)G);
    if ((rc = check_operand(ctx, q, N, H, Lq, D, "cross attention q", &p.q, &p.q_b, &p.q_h, &p.q_l)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, k, N, G, Lk, D, "cross attention k", &p.k, &p.k_b, &p.k_h, &p.k_l)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, v, N, G, Lk, D, "cross attention v", &p.v, &p.v_b, &p.v_h, &p.v_l)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, out, N, H, Lq, D, "cross attention out", &p.out, &p.o_b, &p.o_h, &p.o_l)) != SG_OK) return rc;
    if (out_written && (rc = check_apart(ctx, out, "cross attention out")) != SG_OK) return rc;
    if (mask) {
        if ((rc = sg_check_f32(ctx, mask, "cross attention mask")) != SG_OK) return rc;
        if (mask->rank != 2 || mask->extents[0] != N || mask->extents[1] != Lk) return sg_fail(ctx, SG_ERR_SHAPE, "cross attention mask: expected [%lld, %lld]", (long long)N, (long long)Lk);
        if (Lk > 1 && mask->strides[1] != 1) return sg_fail(ctx, SG_ERR_SHAPE, "cross attention mask: unit stride over the keys expected");
        p.mask = (const float *)mask->base + mask->offset;
        p.mask_b = mask->strides[0];
    }
    if (lse) {
        if ((rc = sg_check_f32(ctx, lse, "cross attention lse")) != SG_OK) return rc;
        if (lse->rank != 3 || lse->extents[0] != N || lse->extents[1] != H || lse->extents[2] != Lq || !sg_is_dense(lse))
            return sg_fail(ctx, SG_ERR_SHAPE, "cross attention lse: expected dense [%lld, %lld, %lld]", (long long)N, (long long)H, (long long)Lq);
        p.lse = (float *)lse->base + lse->offset;
    }
    p.N = (int)N; p.H = (int)H; p.G = (int)G; p.Lq = (int)Lq; p.Lk = (int)Lk;
    return SG_OK;
}

}  // namespace

extern "C" int sg_cross_attention(sg_ctx *ctx, const sg_tensor *q, const sg_tensor *k, const sg_tensor *v, const sg_tensor *mask, float scale,
                                  const sg_tensor *out, const sg_tensor *lse) {
    CrossP p{};
    const int rc = check_call(ctx, q, k, v, mask, out, lse, true, p);
    if (rc != SG_OK) return rc;
    if (!ctx) return SG_ERR_ARG;
    p.o = const_cast<float *>(p.out);
    p.scale = scale;
    sg_device_guard guard(ctx);
    const dim3 grid((unsigned)(p.N * p.H * p.Lq));
    if (q->extents[3] == 64) hipLaunchKernelGGL((cross_forward_kernel<64>), grid, dim3(64), 0, ctx->stream, p);
    else hipLaunchKernelGGL((cross_forward_kernel<32>), grid, dim3(64), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "cross_attention");
    return SG_OK;
}

extern "C" int sg_cross_attention_grad(sg_ctx *ctx, const sg_tensor *q, const sg_tensor *k, const sg_tensor *v, const sg_tensor *mask, float scale,
                                       const sg_tensor *out, const sg_tensor *lse, const sg_tensor *gout, const sg_tensor *gq, const sg_tensor *gk,
                                       const sg_tensor *gv) {
    CrossP p{};
    int rc = check_call(ctx, q, k, v, mask, out, lse, false, p);
    if (rc != SG_OK) return rc;
    if (!lse) return sg_fail(ctx, SG_ERR_ARG, "sg_cross_attention_grad: lse of the forward call expected");
    const int64_t N = p.N, D = q->extents[3];
    const float *ptr;
    if ((rc = check_operand(ctx, gout, N, p.H, p.Lq, D, "sg_cross_attention_grad gout", &p.gout, &p.go_b, &p.go_h, &p.go_l)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, gq, N, p.H, p.Lq, D, "sg_cross_attention_grad gq", &ptr, &p.gq_b, &p.gq_h, &p.gq_l)) != SG_OK) return rc;
    p.gq = const_cast<float *>(ptr);
    if ((rc = check_operand(ctx, gk, N, p.G, p.Lk, D, "sg_cross_attention_grad gk", &ptr, &p.gk_b, &p.gk_h, &p.gk_l)) != SG_OK) return rc;
    p.gk = const_cast<float *>(ptr);
    if ((rc = check_operand(ctx, gv, N, p.G, p.Lk, D, "sg_cross_attention_grad gv", &ptr, &p.gv_b, &p.gv_h, &p.gv_l)) != SG_OK) return rc;
    p.gv = const_cast<float *>(ptr);
    if ((rc = check_apart(ctx, gq, "sg_cross_attention_grad gq")) != SG_OK) return rc;
    if ((rc = check_apart(ctx, gk, "sg_cross_attention_grad gk")) != SG_OK) return rc;
    if ((rc = check_apart(ctx, gv, "sg_cross_attention_grad gv")) != SG_OK) return rc;
    if (!ctx) return SG_ERR_ARG;
    p.scale = scale;
    sg_device_guard guard(ctx);
    const dim3 rows((unsigned)(p.N * p.H * p.Lq)), keys((unsigned)(p.N * p.G * p.Lk));
    if (D == 64) {
        hipLaunchKernelGGL((cross_gq_kernel<64>), rows, dim3(64), 0, ctx->stream, p);
        hipLaunchKernelGGL((cross_gkv_kernel<64>), keys, dim3(64), 0, ctx->stream, p);
    } else {
        hipLaunchKernelGGL((cross_gq_kernel<32>), rows, dim3(64), 0, ctx->stream, p);
        hipLaunchKernelGGL((cross_gkv_kernel<32>), keys, dim3(64), 0, ctx->stream, p);
    }
    SG_CHECK_LAUNCH(ctx, "cross_attention_grad");
    return SG_OK;
}
