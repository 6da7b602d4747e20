// One AdamW step over many parameters, in place, with states in 32 or in 8 bits, for gfx950.
//   m' = beta1 m + (1 - beta1) g;  v' = beta2 v + (1 - beta2) g g
//   value' = value - lr ((m' / (1 - beta1^t)) / (sqrt(v' / (1 - beta2^t)) + eps) + decay value)
// Bound by memory: 28 bytes an element with states in 32 bits, 16 with states in 8, 10 to read the latter.  78.6 M values in 193
// tensors: 390 us (5.6 TB/s), 238 us (5.3 TB/s) and 147 us; a copy of 1 GiB reaches 6.6 TB/s.
//
// 8-bit states.  256 elements share a power of two, so scaling is an addition to exponent fields and exact, and a byte is
// the top of a number's fp32 pattern: no division, no table.  v is never negative and gets the sign's bit for a fifth
// exponent bit: it is a square, and 32 octaves of v are the 16 octaves of g that the 4 exponent bits of m cover.
// Bytes keep 3 mantissa bits (steps of 6 to 12 %), while a step moves v by 1 - beta2 = 0.1 % of what g g is off from it: rounded
// to nearest it would stay where it is for good, unless g g is dozens of times v.  So 16 bits of noise, a hash of element, step
// and seed, are added below the kept bits before the rest is cut off, which rounds up or down with the chances that keep the
// mean.  That holds from the smallest code on: a smaller m is on its way to zero, a smaller v is held at that code (zero would
// make the element's steps as large as eps lets them be).
// The moments are formed without contraction (this file is compiled with -ffp-contract=off): which byte a moment becomes
// hangs on its last bit.
#include "rows.h"

#include <cmath>

namespace {

// Elements per workgroup: 4 wavefronts x 4 blocks of 256, or one block where the step is small and what counts is how long
// one workgroup takes (65 tensors of 210 thousand values: 5.5 us with 4096, 3.7 us with 1024).
constexpr uint32_t chunk_of(bool large) { return large ? 4096 : 1024; }
constexpr uint32_t BLOCK = 256;       // elements that share a scale: 4 for each lane of a wavefront
constexpr int MIN_EXPONENT = 33;      // the smallest number of a block, 31 octaves below its largest, stays normal
constexpr uint32_t V_TOP = 255, M_TOP = 127;

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The tensors of a launch, in its arguments, which may be 4 KB: 100 tensors of 4 pointers, 72 of 6.
template <int POINTERS>
struct Table {
    static constexpr int MAX = POINTERS == 4 ? 100 : 72;
    void *p[MAX][POINTERS];
    uint32_t first_chunk[MAX], n[MAX];  // ~0 and 0 behind the last
};
constexpr int VALUE = 0, GRAD = 1, M = 2, V = 3, M_SCALE = 4, V_SCALE = 5;

struct StepScalars {
    const float *step;
    float lr, beta1, beta2, c1, c2, eps, decay, ln1, ln2;
    uint32_t seed;
};
template <int POINTERS>
struct StepArgs {
    Table<POINTERS> t;
    StepScalars s;
};
static_assert(sizeof(StepArgs<4>) <= 4096 && sizeof(StepArgs<6>) <= 4096, "arguments of a launch");

// The entry a workgroup belongs to: the last one that starts at or before it.  Every lane looks at its own, so the search
// waits once for the arguments, which lie in host memory, and not at every step (65 tensors of 210
// thousand values: two launches of 6.0 us each with a binary search in tables of 56, one of 5.5 us).
template <class T>
__device__ __forceinline__ int find_entry(const T &t, uint32_t chunk) {
    const int lane = threadIdx.x & 63;
    const uint32_t low = t.first_chunk[lane], high = lane < T::MAX - 64 ? t.first_chunk[64 + lane] : ~0u;
    return (int)__popcll(__builtin_amdgcn_ballot_w64(low <= chunk)) + (int)__popcll(__builtin_amdgcn_ballot_w64(high <= chunk)) - 1;
}

// Large steps go past the caches: nothing of them is read again soon.
template <bool NT, class T>
__device__ __forceinline__ T load(const T *p) { return NT ? __builtin_nontemporal_load(p) : *p; }
template <bool NT, class T>
__device__ __forceinline__ void store(T *p, T x) {
    if (NT) __builtin_nontemporal_store(x, p);
    else *p = x;
}

__device__ __forceinline__ bool aligned16(const void *a, const void *b) { return (((uintptr_t)a | (uintptr_t)b) & 15) == 0; }

struct Correction {
    float first, second;  // 1 / (1 - beta1^t), 1 / (1 - beta2^t)
};

// 1 - beta^t as -expm1(t ln beta): for small t the difference would lose what it is made of
__device__ __forceinline__ Correction correction(const StepScalars &a) {
    const float t = *a.step;
    return {-1.0f / expm1f(t * a.ln1), -1.0f / expm1f(t * a.ln2)};
}

__device__ __forceinline__ void step_element(float &value, float g, float &m, float &v, const StepScalars &a, const Correction &c) {
    m = m * a.beta1 + g * a.c1;
    v = v * a.beta2 + g * g * a.c2;
    value = value - a.lr * (m * c.first / (sqrtf(v * c.second) + a.eps) + a.decay * value);
}

template <bool NT>
__global__ void __launch_bounds__(256) adamw_kernel(const StepArgs<4> args) {
    const StepScalars &a = args.s;
    const int entry = find_entry(args.t, blockIdx.x);
    const Correction c = correction(a);
    void *const *p = args.t.p[entry];
    const uint32_t n = args.t.n[entry], base = (blockIdx.x - args.t.first_chunk[entry]) * chunk_of(NT);
    float *xp = (float *)p[VALUE], *mp = (float *)p[M], *vp = (float *)p[V];
    const float *gp = (const float *)p[GRAD];
    const bool vec = aligned16(xp, gp) && aligned16(mp, vp);
#pragma unroll
    for (uint32_t k = 0; k < chunk_of(NT) / 1024; ++k) {
        const uint32_t i = base + k * 1024 + threadIdx.x * 4;
        if (i >= n) return;
        if (vec && i + 4 <= n) {
            f32x4 *x4 = reinterpret_cast<f32x4 *>(xp + i), *m4 = reinterpret_cast<f32x4 *>(mp + i), *v4 = reinterpret_cast<f32x4 *>(vp + i);
            f32x4 x = load<NT>(x4), m = load<NT>(m4), v = load<NT>(v4);
            const f32x4 g = load<NT>(reinterpret_cast<const f32x4 *>(gp + i));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float xj = x[j], mj = m[j], vj = v[j];
                step_element(xj, g[j], mj, vj, a, c);
                x[j] = xj;
                m[j] = mj;
                v[j] = vj;
            }
            store<NT>(x4, x);
            store<NT>(m4, m);
            store<NT>(v4, v);
        } else {
            for (uint32_t j = i; j < i + 4 && j < n; ++j) {
                float x = xp[j], m = mp[j], v = vp[j];
                step_element(x, gp[j], m, v, a, c);
                xp[j] = x;
                mp[j] = m;
                vp[j] = v;
            }
        }
    }
}

__device__ __forceinline__ uint32_t noise(uint32_t i, uint32_t salt) {
    uint32_t h = i * 0x9E3779B9u + salt;
    h = (h ^ (h >> 16)) * 0x82D3099Fu;
    h = (h ^ (h >> 15)) * 0x2ACAE79Fu;
    return h ^ (h >> 16);
}

// e: exponent field of the block's scale; 255 marks a block that holds NaN
__device__ __forceinline__ float decode(uint32_t low, uint32_t e, uint32_t top) {
    if (e == 255) return __builtin_nanf("");
    return low ? __uint_as_float((low + e * 8 + 7 - top) << 20) : 0.0f;
}
__device__ __forceinline__ float decode_m(uint32_t byte, uint32_t e) {
    const float x = decode(byte & 127u, e, M_TOP);
    return byte & 128u ? -x : x;
}

__device__ __forceinline__ uint32_t encode(uint32_t bits, uint32_t noise16, uint32_t e, int top) {
    const int c = (int)((bits + (noise16 << 4)) >> 20) - (int)(e * 8 + 7) + top;
    return (uint32_t)(c < 0 ? 0 : c > top ? top : c);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t y = (uint32_t)__shfl_xor((int)x, o, 64);
        x = x > y ? x : y;
    }
    return x;
}

// exponent field of a block's scale from the largest of its patterns without signs
__device__ __forceinline__ uint32_t scale_exponent(uint32_t largest) {
    const uint32_t e = (largest + 0xFFFFFu) >> 23;
    return e < MIN_EXPONENT ? MIN_EXPONENT : e > 255u ? 255u : e;
}

// A wavefront takes a block of 256 elements, a lane 4 of them and one word of either state.
template <bool NT>
__global__ void __launch_bounds__(256) adamw8_kernel(const StepArgs<6> args) {
    const StepScalars &a = args.s;
    const int entry = find_entry(args.t, blockIdx.x);
    const Correction c = correction(a);
    void *const *p = args.t.p[entry];
    const uint32_t n = args.t.n[entry], chunk = blockIdx.x - args.t.first_chunk[entry];
    float *xp = (float *)p[VALUE], *m_scale = (float *)p[M_SCALE], *v_scale = (float *)p[V_SCALE];
    const float *gp = (const float *)p[GRAD];
    const bool vec = aligned16(xp, gp);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t salt = a.seed + (uint32_t)*a.step * 0xAC502949u;
    uint32_t *mp = (uint32_t *)p[M], *vp = (uint32_t *)p[V];
#pragma unroll
    for (uint32_t k = 0; k < chunk_of(NT) / (4 * BLOCK); ++k) {
        const uint32_t block = chunk * (chunk_of(NT) / BLOCK) + k * 4 + wave;
        if (block * BLOCK >= n) return;  // the whole wavefront
        const uint32_t i = block * BLOCK + lane * 4;
        const uint32_t left = i < n ? (n - i < 4 ? n - i : 4) : 0;
        float x[4] = {}, g[4] = {}, m[4], v[4];
        uint32_t mw = 0, vw = 0;
        if (left == 4 && vec) {
            const f32x4 x4 = load<NT>(reinterpret_cast<const f32x4 *>(xp + i)), g4 = load<NT>(reinterpret_cast<const f32x4 *>(gp + i));
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] = x4[j]; g[j] = g4[j]; }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (j < left) { x[j] = xp[i + j]; g[j] = gp[i + j]; }
        }
        if (left) { mw = load<NT>(mp + i / 4); vw = load<NT>(vp + i / 4); }
        const uint32_t me = __float_as_uint(m_scale[block]) >> 23 & 255u, ve = __float_as_uint(v_scale[block]) >> 23 & 255u;
        uint32_t mtop = 0, vtop = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            m[j] = decode_m(mw >> (8 * j) & 255u, me);
            v[j] = decode(vw >> (8 * j) & 255u, ve, V_TOP);
            step_element(x[j], g[j], m[j], v[j], a, c);
            if (j < left) {
                const uint32_t mb = __float_as_uint(m[j]) & 0x7FFFFFFFu, vb = __float_as_uint(v[j]) & 0x7FFFFFFFu;
                mtop = mtop > mb ? mtop : mb;
                vtop = vtop > vb ? vtop : vb;
            }
        }
        const uint32_t me2 = scale_exponent(wave_max(mtop)), ve2 = scale_exponent(wave_max(vtop));
        mw = vw = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (j >= left) continue;
            const uint32_t h = noise(i + j, salt);
            const uint32_t mb = __float_as_uint(m[j]), vb = __float_as_uint(v[j]) & 0x7FFFFFFFu;
            uint32_t mc = encode(mb & 0x7FFFFFFFu, h & 0xFFFFu, me2, (int)M_TOP);
            if (mc && (mb >> 31)) mc |= 128u;
            uint32_t vc = encode(vb, h >> 16, ve2, (int)V_TOP);
            if (vb && !vc) vc = 1;
            mw |= mc << (8 * j);
            vw |= vc << (8 * j);
        }
        if (left == 4 && vec) store<NT>(reinterpret_cast<f32x4 *>(xp + i), f32x4{x[0], x[1], x[2], x[3]});
        else {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (j < left) xp[i + j] = x[j];
        }
        if (left) { store<NT>(mp + i / 4, mw); store<NT>(vp + i / 4, vw); }
        if (lane == 0) {
            m_scale[block] = __uint_as_float(me2 == 255 ? 0x7FC00000u : me2 << 23);
            v_scale[block] = __uint_as_float(ve2 == 255 ? 0x7FC00000u : ve2 << 23);
        }
    }
}

template <bool NT>
__global__ void __launch_bounds__(256) adamw_state_read_kernel(const Table<6> t) {  // m_out in VALUE's place, v_out in GRAD's
    const int entry = find_entry(t, blockIdx.x);
    void *const *p = t.p[entry];
    const uint32_t n = t.n[entry], base = (blockIdx.x - t.first_chunk[entry]) * chunk_of(NT);
    const uint32_t *mp = (const uint32_t *)p[M], *vp = (const uint32_t *)p[V];
    const float *m_scale = (const float *)p[M_SCALE], *v_scale = (const float *)p[V_SCALE];
    float *mo = (float *)p[VALUE], *vo = (float *)p[GRAD];
    const bool vec = aligned16(mo, vo);
#pragma unroll
    for (uint32_t k = 0; k < chunk_of(NT) / 1024; ++k) {
        const uint32_t i = base + k * 1024 + threadIdx.x * 4;
        if (i >= n) return;
        const uint32_t mw = load<NT>(mp + i / 4), vw = load<NT>(vp + i / 4);
        const uint32_t me = __float_as_uint(m_scale[i / BLOCK]) >> 23 & 255u, ve = __float_as_uint(v_scale[i / BLOCK]) >> 23 & 255u;
        f32x4 m, v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] = decode_m(mw >> (8 * j) & 255u, me);
            v[j] = decode(vw >> (8 * j) & 255u, ve, V_TOP);
        }
        if (vec && i + 4 <= n) {
            store<NT>(reinterpret_cast<f32x4 *>(mo + i), m);
            store<NT>(reinterpret_cast<f32x4 *>(vo + i), v);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (i + j < n) { mo[i + j] = m[j]; vo[i + j] = v[j]; }
        }
    }
}

float *f32_ptr(const sg_tensor *t) { return (float *)t->base + t->offset; }

int check_dense(sg_ctx *ctx, const sg_tensor *t, int dtype, int64_t n, const char *who) {
    const int rc = sg_validate_tensor(ctx, t, who);
    if (rc != SG_OK) return rc;
    if (t->dtype != dtype) return sg_fail(ctx, SG_ERR_DTYPE, "%s: %s expected", who, dtype == SG_FLOAT ? "fp32" : "uint");
    if (!sg_is_dense(t)) return sg_fail(ctx, SG_ERR_SHAPE, "%s: must be dense row-major", who);
    if (n && sg_numel(t) != n) return sg_fail(ctx, SG_ERR_SHAPE, "%s: %lld elements, expected %lld", who, (long long)sg_numel(t), (long long)n);
    return SG_OK;
}

int check_state8(sg_ctx *ctx, const sg_tensor *m, const sg_tensor *v, const sg_tensor *ms, const sg_tensor *vs, int64_t n) {
    int rc;
    if ((rc = check_dense(ctx, m, SG_UINT, (n + 3) / 4, "AdamW first moment")) != SG_OK) return rc;
    if ((rc = check_dense(ctx, v, SG_UINT, (n + 3) / 4, "AdamW second moment")) != SG_OK) return rc;
    if ((rc = check_dense(ctx, ms, SG_FLOAT, (n + BLOCK - 1) / BLOCK, "AdamW first moment's scale")) != SG_OK) return rc;
    return check_dense(ctx, vs, SG_FLOAT, (n + BLOCK - 1) / BLOCK, "AdamW second moment's scale");
}

// Fills one launch's table from tensor `first` on; returns the index behind the last one taken, the workgroups in *chunks.
template <int POINTERS>
int fill_table(Table<POINTERS> &t, uint32_t *chunks, int first, int n_tensors, const sg_tensor *const (&arrays)[6], uint32_t chunk) {
    uint64_t at = 0;
    int i = first, count = 0;
    for (; i < n_tensors && count < Table<POINTERS>::MAX; ++i) {
        const int64_t n = sg_numel(&arrays[VALUE][i]);
        const uint64_t need = ((uint64_t)n + chunk - 1) / chunk;
        if (at + need >= (1ull << 24)) break;  // a launch has fewer than 2^32 threads: the rest in one of its own
        for (int k = 0; k < POINTERS; ++k) t.p[count][k] = f32_ptr(&arrays[k][i]);
        t.n[count] = (uint32_t)n;
        t.first_chunk[count++] = (uint32_t)at;
        at += need;
    }
    for (; count < Table<POINTERS>::MAX; ++count) {
        for (int k = 0; k < POINTERS; ++k) t.p[count][k] = nullptr;
        t.first_chunk[count] = ~0u;
        t.n[count] = 0;
    }
    *chunks = (uint32_t)at;
    return i;
}

// The launches of a step over all tensors, `bytes` an element.
template <int POINTERS, class Launch>
int for_tables(sg_ctx *ctx, int n_tensors, const sg_tensor *const (&arrays)[6], int bytes, Launch launch) {
    int64_t elements = 0;
    for (int i = 0; i < n_tensors; ++i) elements += sg_numel(&arrays[VALUE][i]);
    const bool large = sg_streaming(elements * bytes);
    for (int first = 0; first < n_tensors;) {
        Table<POINTERS> t;
        uint32_t chunks = 0;
        first = fill_table(t, &chunks, first, n_tensors, arrays, chunk_of(large));
        launch(t, chunks, large);
        SG_CHECK_LAUNCH(ctx, "adamw");
    }
    return SG_OK;
}

}  // namespace

extern "C" int sg_adamw_update(sg_ctx *ctx, int n_tensors, const sg_tensor *values, const sg_tensor *grads, const sg_tensor *m, const sg_tensor *v,
                               const sg_tensor *m_scale, const sg_tensor *v_scale, const sg_tensor *step, const sg_adam_hyper *h, uint32_t seed) {
    if (n_tensors < 0) return sg_fail(ctx, SG_ERR_ARG, "sg_adamw_update: %d tensors", n_tensors);
    if (n_tensors && (!values || !grads || !m || !v)) return sg_fail(ctx, SG_ERR_ARG, "sg_adamw_update: null tensor array");
    if (!h || !m_scale != !v_scale) return sg_fail(ctx, SG_ERR_ARG, "sg_adamw_update: %s", h ? "one scale array without the other" : "null scalars");
    if (!(h->beta1 >= 0.0f && h->beta1 < 1.0f && h->beta2 >= 0.0f && h->beta2 < 1.0f)) return sg_fail(ctx, SG_ERR_ARG, "sg_adamw_update: betas must be in [0, 1)");
    int rc;
    if ((rc = check_dense(ctx, step, SG_FLOAT, 1, "sg_adamw_update step")) != SG_OK) return rc;
    const bool eight = m_scale != nullptr;
    // everything is checked before the first launch: a failed call changes nothing
    for (int i = 0; i < n_tensors; ++i) {
        if ((rc = check_dense(ctx, &values[i], SG_FLOAT, 0, "sg_adamw_update value")) != SG_OK) return rc;
        const int64_t n = sg_numel(&values[i]);
        if ((rc = check_dense(ctx, &grads[i], SG_FLOAT, n, "sg_adamw_update grad")) != SG_OK) return rc;
        if (eight) {
            if ((rc = check_state8(ctx, &m[i], &v[i], &m_scale[i], &v_scale[i], n)) != SG_OK) return rc;
        } else {
            if ((rc = check_dense(ctx, &m[i], SG_FLOAT, n, "sg_adamw_update first moment")) != SG_OK) return rc;
            if ((rc = check_dense(ctx, &v[i], SG_FLOAT, n, "sg_adamw_update second moment")) != SG_OK) return rc;
        }
    }
    if (!ctx) return SG_ERR_ARG;
    sg_device_guard guard(ctx);
    StepScalars a{};
    a.step = f32_ptr(step);
    a.lr = h->lr; a.beta1 = h->beta1; a.beta2 = h->beta2; a.c1 = h->one_minus_beta1; a.c2 = h->one_minus_beta2;
    a.eps = h->eps; a.decay = h->weight_decay;
    a.ln1 = (float)std::log((double)h->beta1);
    a.ln2 = (float)std::log((double)h->beta2);
    a.seed = seed;
    const sg_tensor *const arrays[6] = {values, grads, m, v, m_scale, v_scale};
    if (eight)
        return for_tables<6>(ctx, n_tensors, arrays, 16, [&](const Table<6> &t, uint32_t chunks, bool large) {
            if (large) hipLaunchKernelGGL((adamw8_kernel<true>), dim3(chunks), dim3(256), 0, ctx->stream, StepArgs<6>{t, a});
            else hipLaunchKernelGGL((adamw8_kernel<false>), dim3(chunks), dim3(256), 0, ctx->stream, StepArgs<6>{t, a});
        });
    return for_tables<4>(ctx, n_tensors, arrays, 28, [&](const Table<4> &t, uint32_t chunks, bool large) {
        if (large) hipLaunchKernelGGL((adamw_kernel<true>), dim3(chunks), dim3(256), 0, ctx->stream, StepArgs<4>{t, a});
        else hipLaunchKernelGGL((adamw_kernel<false>), dim3(chunks), dim3(256), 0, ctx->stream, StepArgs<4>{t, a});
    });
}

extern "C" int sg_adamw_state_read(sg_ctx *ctx, int n_tensors, const sg_tensor *m, const sg_tensor *v, const sg_tensor *m_scale, const sg_tensor *v_scale,
                                   const sg_tensor *m_out, const sg_tensor *v_out) {
    if (n_tensors < 0) return sg_fail(ctx, SG_ERR_ARG, "sg_adamw_state_read: %d tensors", n_tensors);
    if (n_tensors && (!m || !v || !m_scale || !v_scale || !m_out || !v_out)) return sg_fail(ctx, SG_ERR_ARG, "sg_adamw_state_read: null tensor array");
    int rc;
    for (int i = 0; i < n_tensors; ++i) {
        if ((rc = check_dense(ctx, &m_out[i], SG_FLOAT, 0, "sg_adamw_state_read m_out")) != SG_OK) return rc;
        const int64_t n = sg_numel(&m_out[i]);
        if ((rc = check_dense(ctx, &v_out[i], SG_FLOAT, n, "sg_adamw_state_read v_out")) != SG_OK) return rc;
        if ((rc = check_state8(ctx, &m[i], &v[i], &m_scale[i], &v_scale[i], n)) != SG_OK) return rc;
    }
    if (!ctx) return SG_ERR_ARG;
    sg_device_guard guard(ctx);
    const sg_tensor *const arrays[6] = {m_out, v_out, m, v, m_scale, v_scale};
    return for_tables<6>(ctx, n_tensors, arrays, 10, [&](const Table<6> &t, uint32_t chunks, bool large) {
        if (large) hipLaunchKernelGGL((adamw_state_read_kernel<true>), dim3(chunks), dim3(256), 0, ctx->stream, t);
        else hipLaunchKernelGGL((adamw_state_read_kernel<false>), dim3(chunks), dim3(256), 0, ctx->stream, t);
    });
}
