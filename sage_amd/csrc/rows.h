// Shared by the language-model operators: rows of strided tensors, the context's device, workspaces.
#pragma once
#include "common.h"

// Element offsets of the rows that a tensor's leading axes make, the i-th in row-major order of those axes.
struct sg_rows {
    int rank;
    uint32_t ext[SG_MAX_RANK];
    int64_t st[SG_MAX_RANK];
};

// The first `lead` axes of t, axes that step evenly into one another joined (a dense tensor: one axis); returns their element count.
static inline int64_t sg_make_rows(const sg_tensor *t, int lead, sg_rows *r) {
    int64_t n = 1;
    r->rank = 0;
    for (int i = 0; i < lead; ++i) {
        const int64_t e = t->extents[i], s = t->strides[i];
        n *= e;
        if (e == 1) continue;
        const int k = r->rank;
        if (k > 0 && r->st[k - 1] == s * e) {
            r->ext[k - 1] *= (uint32_t)e;
            r->st[k - 1] = s;
        } else {
            r->ext[k] = (uint32_t)e;
            r->st[k] = s;
            r->rank = k + 1;
        }
    }
    if (r->rank == 0) {
        r->rank = 1;
        r->ext[0] = 1;
        r->st[0] = 0;
    }
    return n;
}

__device__ __forceinline__ int64_t sg_row_offset(const sg_rows &r, uint32_t i) {
    if (r.rank == 1) return (int64_t)i * r.st[0];
    int64_t off = 0;
    for (int k = r.rank - 1; k > 0; --k) {
        const uint32_t q = i / r.ext[k];
        off += (int64_t)(i - q * r.ext[k]) * r.st[k];
        i = q;
    }
    return off + (int64_t)i * r.st[0];
}

// A launch has fewer than 2^32 threads in a dimension.  Grids of more workgroups (of at most 1024 threads) go on in y, and their
// last ones may lie behind the end.
constexpr uint32_t SG_GRID_X = 1u << 21;
static inline dim3 sg_grid(uint64_t workgroups) {
    if (workgroups <= SG_GRID_X) return dim3((unsigned)workgroups);
    return dim3(SG_GRID_X, (unsigned)((workgroups + SG_GRID_X - 1) / SG_GRID_X));
}
__device__ __forceinline__ uint32_t sg_workgroup() { return blockIdx.y * SG_GRID_X + blockIdx.x; }

// Launches go to the device of the context, whichever is current in the calling thread.
struct sg_device_guard {
    int back = -1;
    explicit sg_device_guard(const sg_ctx *ctx) {
        int d = -1;
        if (hipGetDevice(&d) == hipSuccess && d != ctx->device && hipSetDevice(ctx->device) == hipSuccess) back = d;
    }
    ~sg_device_guard() {
        if (back >= 0) (void)hipSetDevice(back);
    }
};

// A workspace of the context's allocator, given back when the call returns: later launches on the context's in-order
// stream may use it again, and a graph that captured the call keeps it (sg_free).
struct sg_workspace {
    sg_ctx *ctx;
    void *p = nullptr;
    explicit sg_workspace(sg_ctx *c) : ctx(c) {}
    sg_workspace(const sg_workspace &) = delete;
    int take(uint64_t bytes) { return sg_alloc(ctx, bytes, &p); }
    ~sg_workspace() {
        if (p) (void)sg_free(ctx, p);
    }
};

// The checks every operand passes: a valid descriptor of the type asked for.
static inline int sg_check_f32(sg_ctx *ctx, const sg_tensor *t, const char *who) {
    const int rc = sg_validate_tensor(ctx, t, who);
    if (rc != SG_OK) return rc;
    if (t->dtype != SG_FLOAT) return sg_fail(ctx, SG_ERR_DTYPE, "%s: fp32 only", who);
    return SG_OK;
}
static inline int sg_check_index(sg_ctx *ctx, const sg_tensor *t, const char *who) {
    const int rc = sg_validate_tensor(ctx, t, who);
    if (rc != SG_OK) return rc;
    if (t->dtype != SG_UINT && t->dtype != SG_INT) return sg_fail(ctx, SG_ERR_DTYPE, "%s: uint or int expected", who);
    return SG_OK;
}
