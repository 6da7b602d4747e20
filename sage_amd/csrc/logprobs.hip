// Log probabilities of given tokens, entropy and top alternatives, and their gradient, for gfx950.
// With c = scale log2(e), m = max x, y_j = (x_j - m) c, s = sum 2^y_j, t = sum 2^y_j y_j over a row's logits x:
//   lse = scale m + ln 2 log2 s;  log p_j = ln 2 (y_j - log2 s);  entropy = ln 2 (log2 s - t / s).
// Bound by memory: the logits are read once (forward), read once and written once (gradient).
//
// Forward: a workgroup a row, or a row over several workgroups where rows are few, whose parts a second launch joins.  A
// thread takes 16 logits a round and keeps (m, s, t) of its own; (m1, s1, t1) moved to a maximum m is
// (m, f s1, f (t1 + s1 d)) with d = (m1 - m) c, f = 2^d.  The k largest come out of the same pass: k lanes' maxima are a
// bound that k logits reach, so a wavefront collects only logits above the k-th largest of its 64 lanes' maxima (a later
// one equal to the bound has a higher index than k that reach it), some ten to a hundred of its share, in a list of its own
// in LDS and without a barrier; the k largest of the wavefronts' lists are ranked at the end.
// 4096 x 30522 without alternatives: 88 us (500 MB, 5.7 TB/s).  1021 x 50257: 39 us without (205 MB, 5.3 TB/s), 48 with 5, 59 with
// 20 (the lists leave room for 4 workgroups a compute unit, which are all rows; what choosing adds no other row's loads hide).
// 4 x 30522 with 5: 9.1 us and a join of 4.6; 4 x 50257 with 64: 23 us and a join of 8.
#include "rows.h"

#include <type_traits>

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any element

constexpr int TOP_MAX = 64;
constexpr int THREADS = 256, VECS = 4, ROUND = THREADS * VECS * 4;  // logits a workgroup takes in a round
constexpr int KEEP = 192;                                           // candidates of a wavefront that wait for the next round
constexpr int LIST = KEEP + 64 * VECS * 4;
constexpr int JOIN = 1024;                                          // candidates of a split row, over all its parts
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
typedef unsigned long long u64;

struct LogpP {
    const float *logits;
    const uint32_t *tokens;
    float *logprob, *entropy, *lse, *top_logprobs;
    uint32_t *top_ids;
    float *part_stats;    // of split rows: [row][split][3]
    unsigned long long *part_keys;  // [row][split][k], 0 where a part has no k logits
    sg_rows rows, token_rows;
    uint32_t R, C, k, splits;
    float scale;
};

// Rising order of the numbers, NaN below all of them, -0 equal to 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t order) { return __uint_as_float((order & 0x80000000u) ? (order & 0x7FFFFFFFu) : ~order); }
__device__ __forceinline__ u64 top_key(float x, uint32_t j) { return ((u64)order_bits(x) << 32) | (uint32_t)~j; }
__device__ __forceinline__ uint32_t index_of(u64 key) { return ~(uint32_t)key; }
__device__ __forceinline__ float value_of(u64 key) { return (key >> 32) ? number_of((uint32_t)(key >> 32)) : __builtin_nanf(""); }

// 0 * -inf is NaN: a distance whose exponential is 0 anyway becomes a finite one; NaN stays
__device__ __forceinline__ float finite(float y) { return y < -1e4f ? -1e4f : y; }

struct Stats {
    float m, s, t;  // m: NaN while no number has been seen
    __device__ float shift() const { return m > -__builtin_inff() ? m : 0.0f; }
    // to the larger maximum m_new (a number, or NaN if there is none still)
    __device__ void move(float m_new, float c) {
        const float to = m_new > -__builtin_inff() ? m_new : 0.0f;
        const float d = s != 0.0f ? finite((m - to) * c) : 0.0f;  // nothing to move yet, whatever m is
        const float f = __builtin_amdgcn_exp2f(d);
        t = f * (t + s * d);
        s = s * f;
        m = m_new;
    }
    // one more logit at distance y; where 2^y is 0 the distance is kept finite, and NaN comes in through the factor
    __device__ void add(float y) {
        const float e = __builtin_amdgcn_exp2f(y);
        s += e;
        t = __builtin_fmaf(e, fmaxf(y, -1e4f), t);
    }
    __device__ void join(float mo, float so, float to, float c) {
        Stats o = {mo, so, to};
        const float top = fmaxf(m, mo);
        move(top, c);
        o.move(top, c);
        s += o.s;
        t += o.t;
    }
};

struct RowResult {
    float shift, log2s, lse, entropy;
    bool empty;  // nothing but -inf
    __device__ RowResult(const Stats &a, float scale) {
        const float inf = __builtin_inff();
        shift = a.shift();
        empty = a.m == -inf && a.s == 0.0f;
        log2s = __builtin_amdgcn_logf(a.s);
        lse = empty ? -inf : __builtin_fmaf(shift, scale, log2s * LN2);
        entropy = empty ? 0.0f : (log2s - a.t / a.s) * LN2;
    }
    // (not by way of base 2, where the distance of the type's lowest value is -inf)
    __device__ float logprob(float x, float scale) const { return empty ? -__builtin_inff() : __builtin_fmaf(x - shift, scale, -(log2s * LN2)); }
};

// The row as 16-byte groups: group g holds logits 4g - lead .. 4g - lead + 3, those that exist.
struct Groups {
    const float *base;
    uint32_t lead, C, count;
    __device__ Groups(const float *x, uint32_t C_) : C(C_) {
        lead = (uint32_t)(((uintptr_t)x & 15) / 4);
        base = x - lead;
        count = (lead + C + 3) / 4;
    }
    // NaN where there is no logit
    __device__ f32x4 load(uint32_t g) const {
        if (4 * g >= lead && 4 * g + 4 <= lead + C) return *reinterpret_cast<const f32x4 *>(base + 4 * g);
        f32x4 v;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) v[j] = 4 * g + j >= lead && 4 * g + j < lead + C ? base[4 * g + j] : __builtin_nanf("");
        return v;
    }
    __device__ bool whole(uint32_t g) const { return 4 * g >= lead && 4 * g + 4 <= lead + C; }
    __device__ bool has(uint32_t g, uint32_t j) const { return 4 * g + j >= lead && 4 * g + j < lead + C; }
    __device__ uint32_t index(uint32_t g, uint32_t j) const { return 4 * g + j - lead; }
};

// The workgroup's Stats: the maximum first, then everyone moves to it once and plain sums are left.
__device__ __forceinline__ Stats block_join(Stats a, float c, float *lds) {  // lds: 12 floats
    float top = a.m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    a.move(top, c);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        a.s += __shfl_xor(a.s, o, 64);
        a.t += __shfl_xor(a.t, o, 64);
    }
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { lds[3 * wave] = a.m; lds[3 * wave + 1] = a.s; lds[3 * wave + 2] = a.t; }
    __syncthreads();
    a = {lds[0], lds[1], lds[2]};
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) a.join(lds[3 * w], lds[3 * w + 1], lds[3 * w + 2], c);
    return a;
}

// A bound (as order_bits) that the k-th largest of the lanes' maxima reaches, its lowest byte cut off; 0 if fewer than k
// lanes have seen a number.
__device__ __forceinline__ uint32_t wave_bound(float lane_max, uint32_t k) {
    const uint32_t mine = order_bits(lane_max), lowest = ~0xFF800000u;  // -inf: the lowest of the numbers
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 8; --bit) {
        const uint32_t higher = bound | (1u << bit);
        if (__popcll(__builtin_amdgcn_ballot_w64(mine >= higher)) >= (int)k) bound = higher;
    }
    return bound == 0 || bound > lowest ? bound : lowest;
}

// Leaves the k largest of a wavefront's n > k keys in front of its list.  They are different, so some bound has exactly k.
__device__ __forceinline__ void wave_select(u64 *list, uint32_t n, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63;
    u64 bound = 0;
    if (n <= 64) {  // a key a lane
        const u64 key = lane < n ? list[lane] : 0;
        for (int bit = 63; bit >= 0; --bit) {
            const u64 higher = bound | (1ull << bit);
            const uint32_t count = (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(key >= higher));
            if (count >= k) bound = higher;
            if (count == k) break;
        }
        const u64 stay = __builtin_amdgcn_ballot_w64(key >= bound && lane < n);
        __builtin_amdgcn_wave_barrier();
        if (stay >> lane & 1) list[__popcll(stay & ((1ull << lane) - 1))] = key;
        __builtin_amdgcn_wave_barrier();
        return;
    }
    constexpr uint32_t EACH = LIST / 64;
    const uint32_t blocks = (n + 63) / 64;
    u64 mine[EACH];  // read once, not for every bit (200 x 50257 with 64 alternatives: 62 us, 78 from LDS)
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i) mine[i] = i < blocks && 64 * i + lane < n ? list[64 * i + lane] : 0;
    for (int bit = 63; bit >= 0; --bit) {
        const u64 higher = bound | (1ull << bit);
        uint32_t count = 0;
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i)
            if (i < blocks) count += (uint32_t)__popcll(__builtin_amdgcn_ballot_w64(mine[i] >= higher));
        if (count >= k) bound = higher;
        if (count == k) break;
    }
    uint32_t to = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (uint32_t i = 0; i < EACH; ++i)
        if (i < blocks) {
            const u64 stay = __builtin_amdgcn_ballot_w64(64 * i + lane < n && mine[i] >= bound);
            if (stay >> lane & 1) list[to + __popcll(stay & ((1ull << lane) - 1))] = mine[i];
            to += (uint32_t)__popcll(stay);
        }
    __builtin_amdgcn_wave_barrier();
}

// Place of a key among n different ones, largest first.
__device__ __forceinline__ uint32_t place_of(const u64 *keys, uint32_t n, u64 key) {
    uint32_t r = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) r += keys[i] > key;
    return r;
}

struct TopLds {
    u64 list[THREADS / 64][LIST];
    uint32_t count[THREADS / 64];
};

template <bool TOP>
__global__ void __launch_bounds__(THREADS) logprobs_kernel(const LogpP p) {
    __shared__ typename std::conditional<TOP, TopLds, uint32_t>::type lds_top;
    __shared__ float lds_stats[12];
    const uint32_t block = sg_workgroup(), row = block / p.splits, split = block - row * p.splits, tid = threadIdx.x;
    if (row >= p.R) return;
    const float *x = p.logits + sg_row_offset(p.rows, row);
    // 16-byte groups at whatever element the row starts; the C % 4 logits behind them are a round of their own
    const uint32_t groups = p.C / 4;
    const uint32_t g0 = (uint32_t)((uint64_t)groups * split / p.splits), g1 = (uint32_t)((uint64_t)groups * (split + 1) / p.splits);
    const float c = p.scale * LOG2E, nan = __builtin_nanf("");
    Stats a = {nan, 0.0f, 0.0f};
    uint32_t bound = 0, n = 0, n_bound = 0;  // of this wavefront: collect above, candidates, candidates when bound was set
    auto collect = [&](float v, uint32_t j, bool take) {
        if constexpr (TOP) {
            const u64 taken = __builtin_amdgcn_ballot_w64(take);
            if (taken == 0) return;
            if (take) lds_top.list[tid >> 6][n + __popcll(taken & ((1ull << (tid & 63)) - 1))] = top_key(v, j);
            n += (uint32_t)__popcll(taken);
        }
    };
    // One round: whole, or with lanes that have no logits left (theirs are NaN).
    auto round = [&](const f32x4 *v, uint32_t g, auto whole) {
        float high = nan;
#pragma unroll
        for (int i = 0; i < VECS; ++i) high = fmaxf(fmaxf(fmaxf(high, v[i].x), v[i].y), fmaxf(v[i].z, v[i].w));
        const float top = fmaxf(a.m, high);
        if (top != a.m) a.move(top, c);
        const float shift = a.shift();
#pragma unroll
        for (int i = 0; i < VECS; ++i)
            if (whole || g + i * THREADS + tid < g1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) a.add((v[i][j] - shift) * c);
            }
        if constexpr (TOP) {
            const bool first = g == g0;
            if (first) bound = wave_bound(a.m, p.k);
            const float limit = number_of(bound);
            // many rounds behind the first have nothing above the bound (where NaN counts, bound is 0)
            if (first || bound == 0 || __builtin_amdgcn_ballot_w64(high > limit) != 0) {
#pragma unroll
                for (int i = 0; i < VECS; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t at = g + i * THREADS + tid;
                        // in the first round also what equals the bound
                        collect(v[i][j], 4 * at + j, (whole || at < g1) && (bound == 0 || (first ? v[i][j] >= limit : v[i][j] > limit)));
                    }
            }
            if (n > KEEP) {
                wave_select(lds_top.list[tid >> 6], n, p.k);
                n = p.k;
            }
            if (n >= n_bound + 16 || first) {
                bound = wave_bound(a.m, p.k);
                n_bound = n;
            }
        }
    };
    auto load = [&](uint32_t at) { return *reinterpret_cast<const f32x4_any *>(x + 4 * (uint64_t)min(at, g1 - 1)); };
    if (g0 < g1) {
        f32x4 next[VECS];
#pragma unroll
        for (int i = 0; i < VECS; ++i) next[i] = load(g0 + i * THREADS + tid);
        uint32_t g = g0;
        for (; g + VECS * THREADS <= g1; g += VECS * THREADS) {
            f32x4 v[VECS];
#pragma unroll
            for (int i = 0; i < VECS; ++i) {
                v[i] = next[i];
                next[i] = load(g + (VECS + i) * THREADS + tid);  // in flight during this round's arithmetic
            }
            round(v, g, std::true_type());
        }
        if (g < g1) {
#pragma unroll
            for (int i = 0; i < VECS; ++i)
                if (g + i * THREADS + tid >= g1) next[i] = f32x4{nan, nan, nan, nan};
            round(next, g, std::false_type());
        }
    }
    if (split == p.splits - 1 && p.C % 4 != 0) {
        const bool there = tid < p.C % 4;
        const float v = there ? x[4 * groups + tid] : nan, top = fmaxf(a.m, v);
        if (there) {
            if (top != a.m) a.move(top, c);
            a.add((v - a.shift()) * c);
        }
        if constexpr (TOP) collect(v, 4 * groups + tid, there && (bound == 0 || v > number_of(bound)));
    }
    const Stats all = block_join(a, c, lds_stats);
    const RowResult r(all, p.scale);
    if (tid == 0) {
        if (p.splits > 1) {
            float *to = p.part_stats + (uint64_t)block * 3;
            to[0] = all.m; to[1] = all.s; to[2] = all.t;
        } else {
            p.lse[row] = r.lse;
            if (p.entropy) p.entropy[row] = r.entropy;
            if (p.logprob) {
                const uint32_t tok = p.tokens[sg_row_offset(p.token_rows, row)];
                p.logprob[row] = tok < p.C ? r.logprob(x[tok], p.scale) : 0.0f;
            }
        }
    }
    if constexpr (TOP) {
        const uint32_t lane = tid & 63, wave = tid >> 6;
        if (n > p.k) wave_select(lds_top.list[wave], n, p.k);
        n = n < p.k ? n : p.k;
        if (lane == 0) lds_top.count[wave] = n;
        __syncthreads();
        if (lane < n) {
            const u64 key = lds_top.list[wave][lane];
            uint32_t at = 0;
            for (int w = 0; w < THREADS / 64; ++w) at += place_of(lds_top.list[w], lds_top.count[w], key);
            if (at < p.k) {
                if (p.splits > 1) p.part_keys[(uint64_t)block * p.k + at] = key;
                else {
                    p.top_ids[(uint64_t)row * p.k + at] = index_of(key);
                    p.top_logprobs[(uint64_t)row * p.k + at] = r.logprob(value_of(key), p.scale);
                }
            }
        }
        if (p.splits > 1) {
            uint32_t all_n = 0;
            for (int w = 0; w < THREADS / 64; ++w) all_n += lds_top.count[w];
            for (uint32_t i = all_n + tid; i < p.k; i += THREADS) p.part_keys[(uint64_t)block * p.k + i] = 0;
        }
    }
}

// Joins the parts of a split row.  (13 parts of 64 candidates: 8 us, 61 us where every candidate is compared with all.)
__global__ void __launch_bounds__(THREADS) logprobs_join_kernel(const LogpP p) {
    __shared__ u64 keys[JOIN], bound;
    __shared__ uint32_t count;
    __shared__ float lds_stats[12];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const float *x = p.logits + sg_row_offset(p.rows, row);
    const float c = p.scale * LOG2E;
    Stats a = {__builtin_nanf(""), 0.0f, 0.0f};
    if (tid < p.splits) {
        const float *from = p.part_stats + ((uint64_t)row * p.splits + tid) * 3;
        a = {from[0], from[1], from[2]};
    }
    const RowResult r(block_join(a, c, lds_stats), p.scale);
    if (tid == 0) {
        p.lse[row] = r.lse;
        if (p.entropy) p.entropy[row] = r.entropy;
        if (p.logprob) {
            const uint32_t tok = p.tokens[sg_row_offset(p.token_rows, row)];
            p.logprob[row] = tok < p.C ? r.logprob(x[tok], p.scale) : 0.0f;
        }
    }
    if (p.k == 0) return;
    const uint32_t n = p.splits * p.k;  // at most JOIN
    const u64 *parts = p.part_keys + (uint64_t)row * n;
    if (n <= 128) {
        if (tid < n) keys[tid] = parts[tid];
        if (tid == 0) count = n;
    } else {
        // A part's keys are in order: the lowest of the parts' ceil(k / splits)-th keys is a bound that k keys reach, and few more do.
        if (tid < 64) {
            u64 low = tid < p.splits ? parts[tid * p.k + (p.k + p.splits - 1) / p.splits - 1] : ~0ull;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 other = __shfl_xor(low, o, 64);
                low = low < other ? low : other;
            }
            if (tid == 0) { bound = low; count = 0; }
        }
        __syncthreads();
        for (uint32_t i = tid; i < n; i += THREADS) {
            const u64 key = parts[i];
            if (key >= bound) keys[atomicAdd(&count, 1u)] = key;  // in any order: each finds its place among all
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i < count; i += THREADS) {
        if (!keys[i]) continue;  // a part with fewer than k logits
        const uint32_t at = place_of(keys, count, keys[i]);
        if (at >= p.k) continue;
        p.top_ids[(uint64_t)row * p.k + at] = index_of(keys[i]);
        p.top_logprobs[(uint64_t)row * p.k + at] = r.logprob(value_of(keys[i]), p.scale);
    }
}

struct LogpGradP {
    const float *logits;
    const uint32_t *tokens;
    const float *lse, *entropy, *g_logprob, *g_entropy;
    float *glogits;
    sg_rows rows, token_rows, gl_rows, ge_rows;
    uint32_t R, C, parts, part;  // workgroups of a row, 16-byte groups of each
    float scale;
};

// lse carries half a step of its own size into every probability: beyond this it is not used (7.6e-6 there).
constexpr float FAR = 128.0f;

// glogits_j = scale (-p_j (gl + ge (log p_j + H)) + [j = token] gl).  4096 x 30522: 182 us (1 GB, 5.5 TB/s; a copy of
// 512 MiB reaches 6.5).  NT: large ones past the caches, 182 us against 207.
template <bool NT>
__global__ void __launch_bounds__(THREADS) logprobs_grad_kernel(const LogpGradP p) {
    __shared__ float lds_stats[12];
    // from the last row to the first: the forward call's last rows are still in the last-level cache
    const uint32_t blocks = p.R * p.parts, from_end = sg_workgroup(), tid = threadIdx.x;
    if (from_end >= blocks) return;
    const uint32_t block = blocks - 1 - from_end, row = block / p.parts, part = block - row * p.parts;
    const float *x = p.logits + sg_row_offset(p.rows, row);
    float *y = p.glogits + (uint64_t)row * p.C;
    const float inf = __builtin_inff(), c = p.scale * LOG2E;
    const float lse = p.lse[row];
    const uint32_t tok = p.g_logprob ? p.tokens[sg_row_offset(p.token_rows, row)] : ~0u;
    const float gl = tok < p.C ? p.g_logprob[sg_row_offset(p.gl_rows, row)] : 0.0f;
    const float ge = p.g_entropy ? p.g_entropy[sg_row_offset(p.ge_rows, row)] : 0.0f;
    const float h = p.g_entropy ? p.entropy[row] : 0.0f;
    // log2 p = (x - shift) c - log2s
    float shift = 0.0f, log2s = lse * LOG2E;
    if (fabsf(lse) > FAR) {  // the row's own maximum and sum again (each workgroup of the row does)
        Stats a = {__builtin_nanf(""), 0.0f, 0.0f};
        for (uint32_t j = tid; j < p.C; j += THREADS) {
            const float v = x[j], top = fmaxf(a.m, v);
            if (top != a.m) a.move(top, c);
            a.s += __builtin_amdgcn_exp2f((v - a.shift()) * c);
        }
        const RowResult r(block_join(a, c, lds_stats), p.scale);
        shift = r.shift;
        log2s = r.log2s;
    }
    auto grad = [&](float v, uint32_t j) {
        // a finite logit may be so low that its distance is not (the type's lowest value hides a token): 0 * -inf is NaN
        const float lp2 = finite((v - shift) * c - log2s);
        const float pr = __builtin_amdgcn_exp2f(lp2);
        float g = -pr * (gl + ge * __builtin_fmaf(lp2, LN2, h));
        if (j == tok) g += gl;
        return v == -inf ? 0.0f : g * p.scale;
    };
    const Groups groups(y, p.C);  // whole groups of the output; the logits of one are at any element
    const uint32_t last = min((part + 1) * p.part, groups.count);
    for (uint32_t g = part * p.part + tid; g < last; g += THREADS) {
        const uint32_t j = groups.index(g, 0);
        if (groups.whole(g)) {
            const f32x4_any *xp = reinterpret_cast<const f32x4_any *>(x + j);
            const f32x4 v = NT ? __builtin_nontemporal_load(xp) : *xp;
            const f32x4 o = {grad(v.x, j), grad(v.y, j + 1), grad(v.z, j + 2), grad(v.w, j + 3)};
            if (NT) __builtin_nontemporal_store(o, reinterpret_cast<f32x4 *>(y + j));
            else *reinterpret_cast<f32x4 *>(y + j) = o;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e)
                if (groups.has(g, e)) y[j + e] = grad(x[j + e], j + e);
        }
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
    // the kernels' scale log2(e) is finite up to here
    if (!(scale > 0.0f && scale <= 0x1p127f)) return sg_fail(ctx, SG_ERR_ARG, "%s: scale must be positive and at most 2^127", who);
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
    // Few rows: a row over several workgroups, at most four for each compute unit in all (what it holds of them), about a
    // round of logits each at least, and no more candidates than a workgroup joins.
    const uint32_t want = 4u * (uint32_t)(ctx->num_cus > 0 ? ctx->num_cus : 256);
    p.splits = want / p.R;
    if (p.splits > (p.C + ROUND - 1) / ROUND) p.splits = (p.C + ROUND - 1) / ROUND;
    if (p.splits > 64) p.splits = 64;
    if (k && p.splits > JOIN / (uint32_t)k) p.splits = JOIN / (uint32_t)k;
    if (p.splits < 1) p.splits = 1;
    sg_device_guard guard(ctx);
    sg_workspace space(ctx);
    if (p.splits > 1) {
        const uint64_t parts = (uint64_t)p.R * p.splits;
        if ((rc = space.take(parts * (8 * k + 12))) != SG_OK) return rc;
        p.part_keys = (unsigned long long *)space.p;
        p.part_stats = (float *)(p.part_keys + parts * k);
    }
    if (k) hipLaunchKernelGGL((logprobs_kernel<true>), sg_grid((uint64_t)p.R * p.splits), dim3(THREADS), 0, ctx->stream, p);
    else hipLaunchKernelGGL((logprobs_kernel<false>), sg_grid((uint64_t)p.R * p.splits), dim3(THREADS), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "token_logprobs");
    if (p.splits > 1) {
        hipLaunchKernelGGL(logprobs_join_kernel, dim3(p.R), dim3(THREADS), 0, ctx->stream, p);
        SG_CHECK_LAUNCH(ctx, "token_logprobs join");
    }
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
    if (f32_ptr(glogits) == f32_ptr(logits) && !sg_is_dense(logits))
        return sg_fail(ctx, SG_ERR_SHAPE, "sg_token_logprobs_grad: in place of logits that are not dense row-major");
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
    // 8192 logits a workgroup: rows of ordinary vocabularies are four or more, so that few rows fill the chip too
    p.part = 2048;
    // (in place: one workgroup a row, which has read the row when it first writes, if it reads the whole row at all)
    if (p.glogits == p.logits) p.part = p.C / 4 + 2;
    p.parts = (p.C + 3 + 4 * p.part - 1) / (4 * p.part);
    sg_device_guard guard(ctx);
    const dim3 grid = sg_grid((uint64_t)p.R * p.parts);
    if (sg_streaming((int64_t)p.R * p.C * 8)) hipLaunchKernelGGL((logprobs_grad_kernel<true>), grid, dim3(THREADS), 0, ctx->stream, p);
    else hipLaunchKernelGGL((logprobs_grad_kernel<false>), grid, dim3(THREADS), 0, ctx->stream, p);
    SG_CHECK_LAUNCH(ctx, "token_logprobs_grad");
    return SG_OK;
}
