// Embedding lookup with scaling and its gradient for gfx950.
//   forward:  out[i, :] = scale * table[id_i, :]            (zeros where id_i is no row of the table)
//   backward: gtable[v, :] = scale * sum_{i: id_i = v} gout[i, :]
// Both are bound by memory: a row is read once and written once.
#include "rows.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct EmbP {
    const float *table;
    const uint32_t *ids;
    float *out;
    sg_rows id_rows;
    uint32_t n, E, V, pieces;
    int64_t table_stride, E_stride;
    float scale;
};

// A wavefront writes 256 columns of one token's row (VEC: 16 bytes a lane): every piece of every row is a wavefront of its
// own, so that the few rows of a serving batch are in flight together too.
template <bool VEC, bool NT>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbP p) {
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= (uint64_t)p.n * p.pieces) return;
    const uint32_t token = (uint32_t)(unit / p.pieces), piece = (uint32_t)(unit - (uint64_t)token * p.pieces);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t id = p.ids[sg_row_offset(p.id_rows, token)];
    const bool known = id < p.V;
    const float *src = p.table + (known ? (int64_t)id * p.table_stride : 0);
    float *dst = p.out + (int64_t)token * p.E;
    if (VEC) {
        const uint32_t c = piece * 256 + lane * 4;
        if (c >= p.E) return;
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (known) v = *reinterpret_cast<const f32x4 *>(src + c) * p.scale;
        if (NT) __builtin_nontemporal_store(v, reinterpret_cast<f32x4 *>(dst + c));
        else *reinterpret_cast<f32x4 *>(dst + c) = v;
    } else {
        for (uint32_t c = piece * 256 + lane; c < p.E && c < piece * 256 + 256; c += 64)
            dst[c] = known ? src[(int64_t)c * p.E_stride] * p.scale : 0.0f;
    }
}

struct EmbGradP {
    const float *gout;
    const uint32_t *ids;
    float *gtable;
    sg_rows id_rows, g_rows;
    uint32_t n, E, V;
    float scale;
};

// One workgroup per table row: it looks through the ids in order and adds the rows of its tokens.
__global__ void __launch_bounds__(256) embedding_grad_kernel(const EmbGradP p) {
    __shared__ uint32_t found[256];
    __shared__ uint32_t count;
    const uint32_t v = blockIdx.x;
    for (uint32_t c0 = 0; c0 < p.E; c0 += 256) {
        const uint32_t c = c0 + threadIdx.x;
        float acc = 0.0f;
        for (uint32_t i0 = 0; i0 < p.n; i0 += 256) {
            __syncthreads();
            const uint32_t i = i0 + threadIdx.x;
            found[threadIdx.x] = i < p.n && p.ids[sg_row_offset(p.id_rows, i)] == v;
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
            if (found[threadIdx.x]) count = 1;
            __syncthreads();
            if (count == 0) continue;
            for (uint32_t j = 0; j < 256; ++j)
                if (found[j] && c < p.E) acc += p.gout[sg_row_offset(p.g_rows, i0 + j) + c];
        }
        if (c < p.E) p.gtable[(int64_t)v * p.E + c] = acc * p.scale;
    }
}

bool aligned16(const void *p) { return ((uintptr_t)p) % 16 == 0; }

// rows [ids.., E] against the ids' extents
int check_rows(sg_ctx *ctx, const sg_tensor *t, const sg_tensor *ids, const char *who) {
    if (t->rank != ids->rank + 1) return sg_fail(ctx, SG_ERR_SHAPE, "%s: rank %d, expected the ids' rank and one axis more", who, t->rank);
    for (int i = 0; i < ids->rank; ++i)
        if (t->extents[i] != ids->extents[i]) return sg_fail(ctx, SG_ERR_SHAPE, "%s: extent[%d] differs from the ids'", who, i);
    return SG_OK;
}

}  // namespace

extern "C" int sg_embedding(sg_ctx *ctx, const sg_tensor *table, const sg_tensor *ids, float scale, const sg_tensor *out) {
    int rc;
    if ((rc = sg_check_f32(ctx, table, "sg_embedding table")) != SG_OK) return rc;
    if ((rc = sg_check_index(ctx, ids, "sg_embedding ids")) != SG_OK) return rc;
    if ((rc = sg_check_f32(ctx, out, "sg_embedding out")) != SG_OK) return rc;
    if (table->rank != 2) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding: table must be [V, E]");
    if ((rc = check_rows(ctx, out, ids, "sg_embedding out")) != SG_OK) return rc;
    const int64_t E = table->extents[1];
    if (out->extents[ids->rank] != E) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding: out's last extent is not the table's");
    if (E > 1 && table->strides[1] != 1) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding: table must have unit stride on its last axis");
    if (!sg_is_dense(out)) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding: out must be dense row-major");
    if (!ctx) return SG_ERR_ARG;
    EmbP p{};
    p.table = (const float *)table->base + table->offset;
    p.ids = (const uint32_t *)ids->base + ids->offset;
    p.out = (float *)out->base + out->offset;
    p.n = (uint32_t)sg_make_rows(ids, ids->rank, &p.id_rows);
    p.E = (uint32_t)E;
    p.V = (uint32_t)table->extents[0];
    p.pieces = (p.E + 255) / 256;
    p.table_stride = table->strides[0];
    p.E_stride = 1;
    p.scale = scale;
    const bool vec = E % 4 == 0 && p.table_stride % 4 == 0 && aligned16(p.table) && aligned16(p.out);
    const bool nt = sg_streaming((int64_t)p.n * E * 4);
    const uint64_t units = (uint64_t)p.n * p.pieces;
    sg_device_guard guard(ctx);
    const dim3 grid((unsigned)((units + 3) / 4));
    if (vec && nt) hipLaunchKernelGGL((embedding_kernel<true, true>), grid, dim3(256), 0, ctx->stream, p);
    else if (vec) hipLaunchKernelGGL((embedding_kernel<true, false>), grid, dim3(256), 0, ctx->stream, p);
    else hipLaunchKernelGGL((embedding_kernel<false, false>), grid, dim3(256), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "embedding");
    return SG_OK;
}

extern "C" int sg_embedding_grad(sg_ctx *ctx, const sg_tensor *gout, const sg_tensor *ids, float scale, const sg_tensor *gtable) {
    int rc;
    if ((rc = sg_check_f32(ctx, gout, "sg_embedding_grad gout")) != SG_OK) return rc;
    if ((rc = sg_check_index(ctx, ids, "sg_embedding_grad ids")) != SG_OK) return rc;
    if ((rc = sg_check_f32(ctx, gtable, "sg_embedding_grad gtable")) != SG_OK) return rc;
    if (gtable->rank != 2) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding_grad: gtable must be [V, E]");
    if ((rc = check_rows(ctx, gout, ids, "sg_embedding_grad gout")) != SG_OK) return rc;
    const int64_t E = gtable->extents[1];
    if (gout->extents[ids->rank] != E) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding_grad: gout's last extent is not the table's");
    if (E > 1 && gout->strides[ids->rank] != 1) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding_grad: gout must have unit stride on its last axis");
    if (!sg_is_dense(gtable)) return sg_fail(ctx, SG_ERR_SHAPE, "sg_embedding_grad: gtable must be dense row-major");
    if (!ctx) return SG_ERR_ARG;
    EmbGradP p{};
    p.gout = (const float *)gout->base + gout->offset;
    p.ids = (const uint32_t *)ids->base + ids->offset;
    p.gtable = (float *)gtable->base + gtable->offset;
    p.n = (uint32_t)sg_make_rows(ids, ids->rank, &p.id_rows);
    (void)sg_make_rows(gout, ids->rank, &p.g_rows);
    p.E = (uint32_t)E;
    p.V = (uint32_t)gtable->extents[0];
    p.scale = scale;
    sg_device_guard guard(ctx);
    hipLaunchKernelGGL(embedding_grad_kernel, dim3(p.V), dim3(256), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "embedding_grad");
    return SG_OK;
}
