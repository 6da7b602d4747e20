// Cross attention of queries to the states of another sequence, forward and backward, fp32 on the CDNA4 matrix cores.
//   forward:  S = c Q K^T over the visible keys, P = e^(S - lse), O = P V, lse = log sum e^S
//   backward: dP = dO V^T, delta = rowsum(dO O), dS = P (dP - delta), dQ = c dS K, dK = c dS^T Q, dV = P^T dO
// The query heads that share a key head are rows below one another: a (batch, key head) pair has R = H/G * Lq rows, row r
// being query r % Lq of head r / Lq of its group, and any number of sharing heads fills the 32-row tiles alike.
//
// Tiles.  A wavefront owns 32 rows (forward, dQ) or 32 keys (dK, dV) and walks the other side in blocks through LDS with
// v_mfma_f32_32x32x2_f32.  What it owns is always the column of the accumulators, lane % 32: score blocks come out as
// S^T (keys x rows) in the forward and dQ kernels and as S (rows x keys) in the dK/dV kernel, with register 4g + s of a
// lane holding index 8g + 4 (lane / 32) + s of the other side, and that is the assignment the next product wants of its
// right operand: P and dS go from accumulators to operands without LDS and without moves between lanes.  Row statistics
// (maximum, sum, lse, delta) are a lane's own in the forward and dQ kernels; hidden keys are a lane's own in the dK/dV
// kernel, where columns do not mix: they are left in and written as zeros.
#include "rows.h"

#include <type_traits>

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any element

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

struct Rows {  // [N, heads, length, D] operand
    const float *p;
    int64_t b, h, l;  // element strides
};

struct CrossP {
    Rows q, k, v, o, go, gq, gk, gv;  // o: written by the forward call, read by the gradient
    const float *mask;
    int *ends;                // of each sequence, one behind its last visible key; NULL: the workgroups look for themselves
    float *lse, *delta;
    float *part_o, *part_ml;  // of split sums: [split][row][D], [split][row][2]
    float *part_k, *part_v;   // [split][key][D]
    int N, H, G, Lq, Lk, R;   // R = H / G * Lq: rows of a (batch, key head) pair
    int64_t mask_b;
    int spread;   // tiles of a pair on all XCDs
    int strided;  // a pair's rows of q and gout lie a stride apart
    float scale;
    uint32_t tiles, pairs, splits;
    sg_fastdiv d_lq, d_tiles, d_pairs, d_g;
};

__device__ __forceinline__ uint32_t fdiv(uint32_t n, sg_fastdiv d) { return (__umulhi(n, d.magic) + n) >> d.shift; }

// One behind the last visible key of a sequence: a padded batch costs what its lengths cost.
__device__ __forceinline__ int visible_end(const CrossP &p, int b, int *lds) {
    if (!p.mask) return p.Lk;
    const float *m = p.mask + b * p.mask_b;
    int end = 0;
    for (int j = threadIdx.x; j < p.Lk; j += 256 * 8) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = m[min(j + 256 * i, p.Lk - 1)];  // in flight together
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (x[i] != 0.0f) end = max(end, min(j + 256 * i, p.Lk - 1) + 1);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) end = max(end, __shfl_xor(end, o, 64));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = end;
    __syncthreads();
    end = max(max(lds[0], lds[1]), max(lds[2], lds[3]));
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(end);
}

__global__ void __launch_bounds__(256) cross_ends_kernel(const CrossP p) {
    __shared__ int lds[4];
    const int end = visible_end(p, blockIdx.x, lds);
    if (threadIdx.x == 0) p.ends[blockIdx.x] = end;
}

struct Work {
    uint32_t split, pair, tile;
    int b, g, end;
};
// Workgroup ids go round-robin over the 8 XCDs.  All tiles of a (split, pair), which share keys or rows, go to one of them,
// and the pairs of a sequence, whose length they have in common, to different ones; where there are few pairs, the tiles go to
// all XCDs (7 x 2 pairs of 1332 rows: both gradients 78 -> 70 us).  Where the lengths are known in front
// (ends), the longest sequences come first: a launch ends when its last workgroup does, and short ones fill the gaps
// (32 x 12 heads of 512 x 512 with lengths 512 to 272: a tenth of the time; 7 x 2 pairs of 1332 rows, 1001 to 501 keys: forward 39
// -> 30 us).  lds: 4 words.
__device__ __forceinline__ Work find_work(const CrossP &p, uint32_t id, int *lds) {
    Work w;
    const uint32_t units = p.pairs * p.splits, even = p.spread ? 0 : units & ~7u;
    uint32_t unit, q;
    if (id < even * p.tiles) {
        q = fdiv(id >> 3, p.d_tiles);
        w.tile = (id >> 3) - q * p.tiles;
        unit = q * 8 + (id & 7);
    } else {
        id -= even * p.tiles;
        q = fdiv(id, p.d_tiles);
        w.tile = id - q * p.tiles;
        unit = even + q;
    }
    // every unit begins with another tile: the workgroups of an XCD go round its shader engines, and tiles behind the last
    // visible key, which are done at once, would all go to the same ones
    w.tile += q - fdiv(q, p.d_tiles) * p.tiles;
    if (w.tile >= p.tiles) w.tile -= p.tiles;
    if (p.spread) {
        w.pair = unit / p.splits;
        w.split = unit - w.pair * p.splits;
    } else {
        w.split = fdiv(unit, p.d_pairs);
        w.pair = unit - w.split * p.pairs;
    }
    w.b = (int)fdiv(w.pair, p.d_g);
    w.g = (int)w.pair - w.b * p.G;
    if (!p.ends) {
        w.end = visible_end(p, w.b, lds);
        return w;
    }
    // the w.b-th longest of the at most 256 sequences
    const int t = threadIdx.x, mine = t < p.N ? p.ends[t] : -1;
    int rank = 0;
    for (int u = 0; u < p.N; ++u) {
        const int e = p.ends[u];
        rank += e > mine || (e == mine && u < t);
    }
    if (t < p.N && rank == w.b) { lds[0] = t; lds[1] = mine; }
    __syncthreads();
    w.b = __builtin_amdgcn_readfirstlane(lds[0]);
    w.end = __builtin_amdgcn_readfirstlane(lds[1]);
    w.pair = (uint32_t)(w.b * p.G + w.g);
    __syncthreads();
    return w;
}

// The same for tiles of KEYS keys, whose work does not depend on the length but is nothing behind it.  Where the lengths are
// known, the tiles that hold visible keys come first, an eighth of them for each XCD, a pair's behind one another, and the
// others, which only write zeros, last: every compute unit gets as many of the former (7 x 2 key heads, 1001 keys, lengths
// 1001 to 501: 57 -> 44 us).  b is -1 for what rounds the grid up to the 8 XCDs.  lds: 8 words.
template <int KEYS>
__device__ __forceinline__ Work find_key_work(const CrossP &p, uint32_t id, int *lds) {
    if (!p.ends) return find_work(p, id, lds);
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6, units = p.G * p.splits, all = units * p.tiles;
    const int mine = t < (uint32_t)p.N ? p.ends[t] : 0;
    const uint32_t count = (uint32_t)((mine + KEYS - 1) / KEYS) * units;
    uint32_t sum = count;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = (uint32_t)__shfl_up((int)sum, o, 64);
        if ((int)lane >= o) sum += y;
    }
    if (lane == 63) lds[wave] = (int)sum;
    if (t == 0) lds[4] = -1;
    __syncthreads();
    uint32_t total = 0, before = sum - count;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (i < wave) before += (uint32_t)lds[i];
        total += (uint32_t)lds[i];
    }
    const uint32_t per = (total + 7) / 8, slot = id >> 3, at = (id & 7) * per + slot;
    const bool first = slot < per && at < total;                   // one with visible keys
    const uint32_t place = first ? at : slot < per ? at - total : id - total;
    const uint32_t from = first ? before : t * all - before, n = first ? count : all - count;
    if (t < (uint32_t)p.N && place >= from && place - from < n) {
        lds[4] = (int)t;
        lds[5] = mine;
        lds[6] = (int)(place - from);
    }
    __syncthreads();
    Work w;
    w.b = __builtin_amdgcn_readfirstlane(lds[4]);
    w.end = __builtin_amdgcn_readfirstlane(lds[5]);
    const uint32_t rest = (uint32_t)__builtin_amdgcn_readfirstlane(lds[6]);
    if (w.b < 0) return w;
    const uint32_t seen = (uint32_t)((w.end + KEYS - 1) / KEYS), tiles = first ? seen : p.tiles - seen, unit = rest / tiles;
    w.tile = rest - unit * tiles + (first ? 0 : seen);
    w.split = unit / (uint32_t)p.G;
    w.g = (int)(unit - w.split * (uint32_t)p.G);
    w.pair = (uint32_t)(w.b * p.G + w.g);
    return w;
}

// Element offset of row r of a pair.
__device__ __forceinline__ int64_t row_at(const CrossP &p, const Rows &x, const Work &w, uint32_t r) {
    const uint32_t hh = fdiv(r, p.d_lq);
    return w.b * x.b + (int64_t)(w.g * (p.H / p.G) + (int)hh) * x.h + (int64_t)(r - hh * p.Lq) * x.l;
}

__device__ __forceinline__ f32x4 load4(const float *p) { return *reinterpret_cast<const f32x4_any *>(p); }
__device__ __forceinline__ void store4(float *p, f32x4 v) { *reinterpret_cast<f32x4_any *>(p) = v; }

// Blocks [first, last) of the `blocks` that this split takes.
__device__ __forceinline__ void split_range(uint32_t blocks, uint32_t split, uint32_t splits, uint32_t *first, uint32_t *last) {
    const uint32_t per = blocks / splits, rest = blocks % splits;
    *first = split * per + (split < rest ? split : rest);
    *last = *first + per + (split < rest ? 1u : 0u);
}

// Tiles of rows in LDS.  Rows lie behind one another without a gap, as loads straight into LDS write them; the 16-byte pieces
// of a row change places with the row's number, so that the 32 rows that a read takes a piece of lie in different banks.
template <int D>
struct Tile {
    static constexpr int PIECES = D / 4;
    __device__ static int turn(int row) { return D == 64 ? row & 15 : (row >> 1) & 7; }
    __device__ static int at(int row, int piece) { return row * D + ((piece ^ turn(row)) << 2); }
};

// One 16-byte piece of a tile.  DMA: straight into LDS, from the wavefront's first lane's piece on, there after arrived();
// needs 16-byte aligned rows.
template <bool DMA>
__device__ __forceinline__ void stage_piece(float *tile, int f, const float *src) {
    if (DMA) {
        float *dst = tile + __builtin_amdgcn_readfirstlane(f & ~63) * 4;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src, (__attribute__((address_space(3))) void *)dst, 16, 0, 0);
    } else {
        *reinterpret_cast<f32x4 *>(tile + f * 4) = load4(src);
    }
}

// Requests ROWS rows of an LDS tile; row_at(r) is where row r begins.
template <int D, int ROWS, bool DMA, class F>
__device__ __forceinline__ void stage(float *tile, F row_at) {
    constexpr int PIECES = Tile<D>::PIECES;
#pragma unroll
    for (int i = 0; i < ROWS * PIECES / 256; ++i) {
        const int f = i * 256 + (int)threadIdx.x, row = f / PIECES;
        stage_piece<DMA>(tile, f, row_at(row) + ((f % PIECES) ^ Tile<D>::turn(row)) * 4);
    }
}

// The same of rows that lie a stride apart.  A thread's pieces are 1024 / D rows apart and in the same place of each, so what
// is its own of their addresses is fixed for the kernel; in 32 bits (DMA: strides below 2^22 elements) beside a base in scalar
// registers, the loads need no vector instruction, which would be taken from the matrix pipes' time.
template <int D>
struct Strided {
    static constexpr int STEP = 1024 / D;
    const float *x;
    int64_t l;
    int total, row, wave_piece;
    uint32_t own;  // bytes from a tile's first row to this thread's first piece
    __device__ Strided(const float *x_, int64_t l_, int total_) : x(x_), l(l_), total(total_) {
        row = (int)threadIdx.x / Tile<D>::PIECES;
        own = ((uint32_t)row * (uint32_t)l + (((int)threadIdx.x % Tile<D>::PIECES) ^ Tile<D>::turn(row)) * 4) * 4;
        wave_piece = __builtin_amdgcn_readfirstlane((int)threadIdx.x & ~63);
    }
    template <int ROWS, bool DMA>
    __device__ __forceinline__ void stage(float *tile, int first) const {
        const bool whole = first + ROWS <= total;
#pragma unroll
        for (int i = 0; i < ROWS / STEP; ++i) {
            if (DMA) {
                const char *base = reinterpret_cast<const char *>(x + (int64_t)(whole ? first + i * STEP : first) * l);
                uint32_t at = own;
                // rows past the end repeat the last one
                if (!whole) at += (uint32_t)(min(row + i * STEP, total - 1 - first) - row) * (uint32_t)l * 4;
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(base + at),
                                                 (__attribute__((address_space(3))) void *)(tile + (i * 256 + wave_piece) * 4), 16, 0, 0);
            } else {
                const int64_t r = min(first + i * STEP + row, total - 1);
                const float *src = x + r * l + (((int)threadIdx.x % Tile<D>::PIECES) ^ Tile<D>::turn(row)) * 4;
                *reinterpret_cast<f32x4 *>(tile + (i * 256 + (int)threadIdx.x) * 4) = load4(src);
            }
        }
    }
};
// What this wavefront requested is in LDS (and in registers).
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Zeros in place of the rows whose bit is not set, by the threads that staged them: 0 * NaN is NaN.
template <int D, int ROWS>
__device__ __forceinline__ void clear_rows(float *tile, const uint32_t *seen) {
    constexpr int PIECES = Tile<D>::PIECES;
#pragma unroll
    for (int i = 0; i < ROWS * PIECES / 256; ++i) {
        const int f = i * 256 + (int)threadIdx.x, row = f / PIECES;
        uint32_t word = seen[0];
#pragma unroll
        for (int k = 1; k < ROWS / 32; ++k) word = row / 32 == k ? seen[k] : word;
        if (!(word >> (row % 32) & 1)) *reinterpret_cast<f32x4 *>(tile + f * 4) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// Which keys of a block are visible, as bits: requested with the block, the same in every wavefront.
template <int KB>
struct Visible {
    static constexpr int N = (KB + 63) / 64;
    float x[N];  // as loaded: nothing looks at it, and waits for it, before bits()
    __device__ static int key(int i) { return i * 64 + ((int)threadIdx.x & (KB < 64 ? KB - 1 : 63)); }
    // mask: any 32 readable floats where there is none
    __device__ void request(const float *mask, bool is_mask, int j0, int Lk) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = mask[is_mask ? min(j0 + key(i), Lk - 1) : key(i) & 31];
    }
    __device__ bool bits(bool is_mask, int j0, int Lk, uint32_t *words) const {  // whether all are
        bool all = true;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint64_t b = __builtin_amdgcn_ballot_w64((!is_mask || x[i] != 0.0f) && j0 + key(i) < Lk);
            words[KB < 64 ? 0 : 2 * i] = (uint32_t)b;
            if (KB >= 64) words[2 * i + 1] = (uint32_t)(b >> 32);
            all = all && b == ~0ull;
        }
        return all;
    }
};

// A wavefront's own 32 columns as the right operand: register [g][s] of lane (c, h) = x[c][8g + 4h + s].  Loaded from memory
// as they are needed, 32 bytes of 32 rows an instruction: a way through LDS would take whole lines, but one wait more in
// front of the first block, and the buffers that this block is on its way into.
template <int D>
struct Own {
    f32x4 x[D / 8];
    __device__ void load(const float *row, int h) {
#pragma unroll
        for (int g = 0; g < D / 8; ++g) x[g] = load4(row + 8 * g + 4 * h);
    }
    __device__ void scale(float f) {
#pragma unroll
        for (int g = 0; g < D / 8; ++g) x[g] *= f;
    }
};

__device__ __forceinline__ floatx16 zero16() {
    floatx16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.0f;
    return z;
}

// 32 rows of an LDS tile times a wavefront's own columns, contracted over the head dimension.
template <int D>
__device__ __forceinline__ floatx16 scores(const float *tile, const Own<D> &own, int c, int h) {
    floatx16 acc = zero16();
#pragma unroll
    for (int g = 0; g < D / 8; ++g) {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(&tile[Tile<D>::at(c, 2 * g + h)]);
#pragma unroll
        for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s], own.x[g][s], acc, 0, 0, 0);
    }
    return acc;
}

// acc[j] += tile^T . w over the tile's 32 rows.  Row m of output block j stands for head index ND m + j, so that what a
// lane feeds to the ND blocks for one row is adjacent in LDS.
template <int D>
__device__ __forceinline__ void accumulate(const float *tile, const floatx16 &w, floatx16 *acc, int c, int h) {
    constexpr int ND = D / 32;
    typedef float vecND __attribute__((ext_vector_type(ND)));
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        vecND a[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) a[s] = *reinterpret_cast<const vecND *>(&tile[Tile<D>::at(8 * g + 4 * h + s, ND * c / 4) + ND * c % 4]);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < ND; ++j) acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s][j], w[4 * g + s], acc[j], 0, 0, 0);
    }
}

// What accumulate() left of column c: consecutive head indices ND (8g + 4h) .. + 4 ND, times f.
template <int D>
__device__ __forceinline__ void write_column(float *row, const floatx16 *acc, float f, int h) {
    constexpr int ND = D / 32;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float t[4 * ND];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < ND; ++j) t[ND * s + j] = acc[j][4 * g + s] * f;
#pragma unroll
        for (int c = 0; c < ND; ++c) store4(row + ND * (8 * g + 4 * h) + 4 * c, f32x4{t[4 * c], t[4 * c + 1], t[4 * c + 2], t[4 * c + 3]});
    }
}

// Walks the visible blocks of KB keys, two LDS buffers in turn: while one is worked on, the next block is on its way into
// the other, and there is one barrier a block.  (The buffers are arrays of their own: the compiler waits for a load into LDS
// in front of any read that it cannot tell from the load's target.)  ready() is called when the first block is on its way;
// work(keys' tile, values' tile, bits of this wavefront's 32 keys).
template <int D, int KB, bool DMA, class G, class F>
__device__ __forceinline__ void walk_keys(const CrossP &p, const Work &w, float (&lds0)[2 * KB * D], float (&lds1)[2 * KB * D], uint32_t first, uint32_t last, int kw,
                                          G ready, F work) {
    const float *K = p.k.p + w.b * p.k.b + w.g * p.k.h, *V = p.v.p + w.b * p.v.b + w.g * p.v.h;
    const bool is_mask = p.mask != nullptr;
    const float *mask = is_mask ? p.mask + w.b * p.mask_b : K;
    Visible<KB> next;
    const Strided<D> keys(K, p.k.l, p.Lk), values(V, p.v.l, p.Lk);
    auto request = [&](uint32_t blk, float *to) {
        const int j0 = (int)blk * KB;
        keys.template stage<KB, DMA>(to, j0);
        values.template stage<KB, DMA>(to + KB * D, j0);
        next.request(mask, is_mask, j0, p.Lk);
    };
    auto step = [&](uint32_t blk, float *tile, float *other) {
        arrived();
        uint32_t seen[(KB + 31) / 32];
        if (!next.bits(is_mask, (int)blk * KB, p.Lk, seen)) {
            clear_rows<D, KB>(tile, seen);
            clear_rows<D, KB>(tile + KB * D, seen);
        }
        __syncthreads();
        if (blk + 1 < last) request(blk + 1, other);
        uint32_t mine = seen[0];
#pragma unroll
        for (int k = 1; k < KB / 32; ++k) mine = kw == k * 32 ? seen[k] : mine;
        work(tile + kw * D, tile + (KB + kw) * D, (uint32_t)__builtin_amdgcn_readfirstlane((int)mine));
    };
    if (first < last) request(first, lds0);
    ready();
    for (uint32_t blk = first; blk < last; blk += 2) {
        step(blk, lds0, lds1);
        if (blk + 1 < last) step(blk + 1, lds1, lds0);
    }
}

// Merges accumulators through LDS: wavefronts RW and up hand theirs over, the first RW call join(slot) for each.
template <int RW, int SLOT, class G, class J>
__device__ __forceinline__ bool merge_waves(float *lds, int wave, int lane, G give, J join) {
    constexpr int KW = 4 / RW;
    if (KW == 1) return true;
    __syncthreads();
    if (wave >= RW) give(&lds[((wave - RW) * 64 + lane) * SLOT]);
    __syncthreads();
    if (wave >= RW) return false;
#pragma unroll
    for (int o = 1; o < KW; ++o) join(&lds[((o - 1) * RW * 64 + wave * 64 + lane) * SLOT]);
    return true;
}

// ---- forward.  RW wavefronts take the workgroup's 32 RW rows, the 4 / RW times as many share each block's keys and are
// merged through LDS at the end.  Bound by the matrix pipes, which fp32 vector instructions share: counters show them busy for
// 84 % (D = 64) and 77 % (D = 32) of the time a compute unit has work, the vector instructions of the softmax are the rest.
// 32 x 12 heads, 512 x 512, D = 64: 224 us (115 TFLOP/s); lengths 512 to 272: 181 us; D = 32: 126 us (102 TFLOP/s).
template <int D, int RW, bool DMA>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(RW == 4 ? 3 : 1))) cross_forward_kernel(const CrossP p) {
    constexpr int KW = 4 / RW, KB = 32 * KW, ND = D / 32, SLOT = 16 * ND + 2;
    __shared__ __attribute__((aligned(16))) float lds0[2 * KB * D], lds1[2 * KB * D];  // two buffers of keys and values
    __shared__ int lds_end[4];
    static_assert((KW - 1) * RW * 64 * SLOT <= 2 * KB * D, "the merge fits in a buffer");
    const Work w = find_work(p, blockIdx.x, lds_end);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 31, h = lane >> 5;
    const uint32_t r = w.tile * (32 * RW) + (wave % RW) * 32 + c;
    const float inf = __builtin_inff();
    Own<D> q;
    q.load(p.q.p + row_at(p, p.q, w, min(r, (uint32_t)p.R - 1)), h);  // a row past the end repeats the last one; it is not written
    floatx16 acc[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j] = zero16();
    float m_run = -inf, l_run = 0.0f, shift = 0.0f;
    uint32_t first, last;
    split_range((w.end + KB - 1) / KB, w.split, p.splits, &first, &last);
    walk_keys<D, KB, DMA>(p, w, lds0, lds1, first, last, wave / RW * 32, [&] { q.scale(p.scale * LOG2E); /* scores are logarithms to base 2 */ },
                          [&](const float *kt, const float *vt, uint32_t seen) {
        floatx16 s = scores<D>(kt, q, c, h);
        if (seen != ~0u) {
            const uint32_t mine = seen >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!(mine >> (8 * (r / 4) + r % 4) & 1)) s[r] = -inf;
        }
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        // The largest so far and 8 (octaves) more is what exponentials are taken relative to: later blocks rarely pass it and
        // have everything moved to a new one.
        if (__builtin_amdgcn_ballot_w64(top > m_run) != 0) {
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float m_new = top > m_run ? top + 8.0f : m_run;
            shift = m_new == -inf ? 0.0f : m_new;  // nothing visible so far: every exponential below is 0
            const float f = __builtin_amdgcn_exp2f(m_run - shift);
            l_run *= f;
#pragma unroll
            for (int j = 0; j < ND; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[j][r] *= f;
            m_run = m_new;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(s[r] - shift);
            l_run += s[r];
        }
        accumulate<D>(vt, s, acc, c, h);
    });
    l_run += __shfl_xor(l_run, 32, 64);
    const bool writes = merge_waves<RW, SLOT>(lds0, wave, lane, [&](float *to) {
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) to[16 * j + r] = acc[j][r];
        to[16 * ND] = m_run;
        to[16 * ND + 1] = l_run;
    }, [&](const float *from) {
        const float mo = from[16 * ND], m = fmaxf(m_run, mo), shift = m == -inf ? 0.0f : m;
        const float fa = __builtin_amdgcn_exp2f(m_run - shift), fb = __builtin_amdgcn_exp2f(mo - shift);
        l_run = l_run * fa + from[16 * ND + 1] * fb;
        m_run = m;
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[j][r] = acc[j][r] * fa + from[16 * j + r] * fb;
    });
    if (!writes || r >= (uint32_t)p.R) return;
    const int64_t row = (int64_t)w.pair * p.R + r;
    if (p.splits > 1) {
        const int64_t at = (int64_t)w.split * p.pairs * p.R + row;
        write_column<D>(p.part_o + at * D, acc, 1.0f, h);
        if (h == 0) { p.part_ml[2 * at] = m_run; p.part_ml[2 * at + 1] = l_run; }
        return;
    }
    write_column<D>(const_cast<float *>(p.o.p) + row_at(p, p.o, w, r), acc, l_run == 0.0f ? 0.0f : 1.0f / l_run, h);
    if (p.lse && h == 0) p.lse[row] = l_run == 0.0f ? -inf : (m_run + __builtin_amdgcn_logf(l_run)) * LN2;
}

// ---- forward with up to 8 rows a pair (a serving step).  Bound by memory: K and V are read once for few products, on
// the vector unit.  D / 4 lanes hold a key's 16-byte pieces, so a wavefront takes 4 or 8 keys an instruction; every group of
// lanes runs a softmax of its own over its keys, merged at the end.  UNROLL keys a group are in flight behind the UNROLL
// that are worked on.  One query of 32 x 12 heads over 512 to 272 keys of size 64: 17.4 us (75 MB, 4.3 TB/s).
template <int D>
__device__ __forceinline__ float group_sum(float x) {  // over the D / 4 lanes of a key, in all of them
    auto move = [](float v, auto ctrl) { return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), decltype(ctrl)::value, 0xF, 0xF, true)); };
    x += move(x, std::integral_constant<int, 0xB1>());   // quad_perm 1 0 3 2
    x += move(x, std::integral_constant<int, 0x4E>());   // quad_perm 2 3 0 1
    x += move(x, std::integral_constant<int, 0x141>());  // row_half_mirror
    if (D == 64) x += move(x, std::integral_constant<int, 0x140>());  // row_mirror
    return x;
}

template <int D, int ROWS, int UNROLL>
__global__ void __launch_bounds__(256) cross_few_kernel(const CrossP p) {
    constexpr int LPK = D / 4, KEYS = 64 / LPK, STEP = KEYS * UNROLL;  // lanes a key, keys an instruction, keys a step
    __shared__ int lds_end[4];
    __shared__ float lds_ml[4][ROWS][2];
    __shared__ __attribute__((aligned(16))) float lds_o[4][ROWS][D];
    const Work w = find_work(p, blockIdx.x, lds_end);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / LPK, col = lane % LPK * 4;
    const float *K = p.k.p + w.b * p.k.b + w.g * p.k.h + col, *V = p.v.p + w.b * p.v.b + w.g * p.v.h + col;
    const float *mask = p.mask ? p.mask + w.b * p.mask_b : nullptr;
    const float inf = __builtin_inff(), c2 = p.scale * LOG2E;
    f32x4 q[ROWS], acc[ROWS];
    float m[ROWS], l[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        q[r] = load4(p.q.p + row_at(p, p.q, w, min(r, p.R - 1)) + col) * c2;
        acc[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        m[r] = -inf;
        l[r] = 0.0f;
    }
    const int end = w.end;
    uint32_t first, last;
    split_range((end + STEP - 1) / STEP, w.split, p.splits, &first, &last);
    f32x4 kn[UNROLL], vn[UNROLL];
    float mn[UNROLL];
    auto request = [&](uint32_t step) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = (int)step * STEP + u * KEYS + sub, at = min(j, p.Lk - 1);
            kn[u] = load4(K + (int64_t)at * p.k.l);
            vn[u] = load4(V + (int64_t)at * p.v.l);
            mn[u] = j < end ? (mask ? mask[at] : 1.0f) : 0.0f;
        }
    };
    if (first + wave < last) request(first + wave);
    for (uint32_t step = first + wave; step < last; step += 4) {
        f32x4 k[UNROLL], v[UNROLL];
        bool seen[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            k[u] = kn[u];
            seen[u] = mn[u] != 0.0f;
            v[u] = seen[u] ? vn[u] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};  // 0 * NaN is NaN
        }
        if (step + 4 < last) request(step + 4);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            float s[UNROLL], top = m[r];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const float d = __builtin_fmaf(q[r].w, k[u].w, __builtin_fmaf(q[r].z, k[u].z, __builtin_fmaf(q[r].y, k[u].y, q[r].x * k[u].x)));
                s[u] = seen[u] ? group_sum<D>(d) : -inf;
                top = fmaxf(top, s[u]);
            }
            const float shift = top == -inf ? 0.0f : top;
            if (__builtin_amdgcn_ballot_w64(top != m[r]) != 0) {
                const float f = __builtin_amdgcn_exp2f(m[r] - shift);
                l[r] *= f;
                acc[r] *= f;
                m[r] = top;
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const float e = __builtin_amdgcn_exp2f(s[u] - shift);
                l[r] += e;
                acc[r] += v[u] * e;
            }
        }
    }
    // the lane groups of a wavefront, then the wavefronts
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        float top = m[r];
#pragma unroll
        for (int o = LPK; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float f = __builtin_amdgcn_exp2f(m[r] - (top == -inf ? 0.0f : top));
        l[r] *= f;
        acc[r] *= f;
#pragma unroll
        for (int o = LPK; o < 64; o <<= 1) {
            l[r] += __shfl_xor(l[r], o, 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[r][j] += __shfl_xor(acc[r][j], o, 64);
        }
        if (sub == 0) *reinterpret_cast<f32x4 *>(&lds_o[wave][r][col]) = acc[r];
        if (lane == 0) { lds_ml[wave][r][0] = top; lds_ml[wave][r][1] = l[r]; }
    }
    __syncthreads();
    if ((int)threadIdx.x >= ROWS * LPK) return;
    const int r = threadIdx.x / LPK, c = threadIdx.x % LPK * 4;
    if (r >= p.R) return;
    float top = -inf, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, lds_ml[i][r][0]);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float f = __builtin_amdgcn_exp2f(lds_ml[i][r][0] - (top == -inf ? 0.0f : top));
        sum += lds_ml[i][r][1] * f;
        o += *reinterpret_cast<const f32x4 *>(&lds_o[i][r][c]) * f;
    }
    const int64_t row = (int64_t)w.pair * p.R + r;
    if (p.splits > 1) {
        const int64_t at = (int64_t)w.split * p.pairs * p.R + row;
        *reinterpret_cast<f32x4 *>(p.part_o + at * D + c) = o;
        if (c == 0) { p.part_ml[2 * at] = top; p.part_ml[2 * at + 1] = sum; }
        return;
    }
    store4(const_cast<float *>(p.o.p) + row_at(p, p.o, w, r) + c, o * (sum == 0.0f ? 0.0f : 1.0f / sum));
    if (p.lse && c == 0) p.lse[row] = sum == 0.0f ? -inf : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// Joins the splits of a row: D / 4 lanes a row (bound by its launch: 4 to 8 us).
template <int D>
__global__ void __launch_bounds__(256) cross_join_kernel(const CrossP p) {
    constexpr int LPR = D / 4;
    const uint32_t total = p.pairs * p.R, row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, col = threadIdx.x % LPR * 4;
    if (row >= total) return;
    const float inf = __builtin_inff();
    float m = -inf, l = 0.0f;
    for (uint32_t i = 0; i < p.splits; ++i) m = fmaxf(m, p.part_ml[2 * ((int64_t)i * total + row)]);
    const float shift = m == -inf ? 0.0f : m;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t i = 0; i < p.splits; ++i) {
        const int64_t at = (int64_t)i * total + row;
        const float f = __builtin_amdgcn_exp2f(p.part_ml[2 * at] - shift);
        l += p.part_ml[2 * at + 1] * f;
        acc += *reinterpret_cast<const f32x4 *>(p.part_o + at * D + col) * f;
    }
    Work w;
    w.pair = row / p.R;
    w.b = (int)fdiv(w.pair, p.d_g);
    w.g = (int)w.pair - w.b * p.G;
    store4(const_cast<float *>(p.o.p) + row_at(p, p.o, w, row - w.pair * p.R) + col, acc * (l == 0.0f ? 0.0f : 1.0f / l));
    if (p.lse && col == 0) p.lse[row] = l == 0.0f ? -inf : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// ---- gradient of the queries (and delta, for the other kernel).  Three products a block, the matrix pipes busy for 84 % of the
// time there is work.  32 x 12 heads, 512 x 512, D = 64: 329 us (117 TFLOP/s); lengths 512 to 272: 265 us.
// GIVEN: delta is there already.
template <int D, int RW, bool DMA, bool GIVEN>
__device__ __forceinline__ void gq_work(const CrossP &p, uint32_t id, float (&lds0)[256 / RW * D], float (&lds1)[256 / RW * D], int *lds_end) {
    constexpr int KW = 4 / RW, KB = 32 * KW, ND = D / 32, SLOT = 16 * ND;
    static_assert((KW - 1) * RW * 64 * SLOT <= 2 * KB * D, "the merge fits in a buffer");
    const Work w = find_work(p, id, lds_end);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 31, h = lane >> 5;
    const uint32_t r = w.tile * (32 * RW) + (wave % RW) * 32 + c, rr = min(r, (uint32_t)p.R - 1);
    const int64_t row = (int64_t)w.pair * p.R + rr;
    Own<D> q, go, o;
    q.load(p.q.p + row_at(p, p.q, w, rr), h);
    go.load(p.go.p + row_at(p, p.go, w, rr), h);
    if (!GIVEN) o.load(p.o.p + row_at(p, p.o, w, rr), h);
    float lse2 = p.lse[row], delta = GIVEN ? p.delta[row] : 0.0f;
    floatx16 acc[ND];
#pragma unroll
    for (int j = 0; j < ND; ++j) acc[j] = zero16();
    uint32_t first, last;
    split_range((w.end + KB - 1) / KB, w.split, p.splits, &first, &last);
    walk_keys<D, KB, DMA>(p, w, lds0, lds1, first, last, wave / RW * 32, [&] {
        q.scale(p.scale * LOG2E);
        lse2 *= LOG2E;
        if (GIVEN) return;
#pragma unroll
        for (int g = 0; g < D / 8; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i) delta += o.x[g][i] * go.x[g][i];
        delta += __shfl_xor(delta, 32, 64);
        if (w.split == 0 && wave < RW && h == 0 && r < (uint32_t)p.R) p.delta[row] = delta;
    }, [&](const float *kt, const float *vt, uint32_t seen) {
        floatx16 s = scores<D>(kt, q, c, h);
        const floatx16 dp = scores<D>(vt, go, c, h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] - lse2) * (dp[i] - delta);
        if (seen != ~0u) {
            const uint32_t mine = seen >> (4 * h);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!(mine >> (8 * (i / 4) + i % 4) & 1)) s[i] = 0.0f;
        }
        accumulate<D>(kt, s, acc, c, h);
    });
    const bool writes = merge_waves<RW, SLOT>(lds0, wave, lane, [&](float *to) {
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) to[16 * j + i] = acc[j][i];
    }, [&](const float *from) {
#pragma unroll
        for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j][i] += from[16 * j + i];
    });
    if (!writes || r >= (uint32_t)p.R) return;
    if (p.splits > 1) write_column<D>(p.part_o + ((int64_t)w.split * p.pairs * p.R + row) * D, acc, p.scale, h);
    else write_column<D>(const_cast<float *>(p.gq.p) + row_at(p, p.gq, w, r), acc, p.scale, h);
}

template <int D, int RW, bool DMA>
__global__ void __launch_bounds__(256) cross_gq_kernel(const CrossP p) {
    __shared__ __attribute__((aligned(16))) float lds0[256 / RW * D], lds1[256 / RW * D];
    __shared__ int lds_end[4];
    gq_work<D, RW, DMA, false>(p, blockIdx.x, lds0, lds1, lds_end);
}

// ---- gradients of keys and values: a wavefront owns 32 keys and walks the rows of the pair, 32 at a time.  CW wavefronts
// take the workgroup's 32 CW keys, the 4 / CW times as many share each block's rows and are added up through LDS.  Four
// products a block, the matrix pipes busy for 86 %.  32 x 12 heads, 512 x 512, D = 64: 431 us (119 TFLOP/s); lengths 512 to 272:
// 379 us.  (dQ from here too would save two of the seven products of a gradient, and cost sums over workgroups.)
template <int D, int CW, bool DMA>
__device__ __forceinline__ void gkv_work(const CrossP &p, uint32_t id, float (&lds0)[256 / CW * D], float (&lds1)[256 / CW * D], float (&rows0)[256 / CW],
                                         float (&rows1)[256 / CW], int *lds_end) {  // rows: their lse and delta
    constexpr int GW = 4 / CW, RB = 32 * GW, ND = D / 32, KEYS = 32 * CW, SLOT = 32 * ND;
    static_assert((GW - 1) * CW * 64 * SLOT <= 2 * RB * D, "the merge fits in a buffer");
    const Work w = find_key_work<KEYS>(p, id, lds_end);
    if (w.b < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 31, h = lane >> 5;
    const int j0 = (int)w.tile * KEYS, j = j0 + (wave % CW) * 32 + c, rw = wave / CW * 32;
    const float *K = p.k.p + w.b * p.k.b + w.g * p.k.h, *V = p.v.p + w.b * p.v.b + w.g * p.v.h;
    const bool seen = j < w.end && (!p.mask || p.mask[w.b * p.mask_b + j] != 0.0f);
    const float inf = __builtin_inff();
    floatx16 gk[ND], gv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) gk[d] = gv[d] = zero16();
    if (j0 < w.end) {
        Own<D> k, v;  // k scaled in front of the walk: scores are logarithms to base 2
        k.load(K + (int64_t)min(j, p.Lk - 1) * p.k.l, h);
        v.load(V + (int64_t)min(j, p.Lk - 1) * p.v.l, h);
        float lreg = 0.0f, dreg = 0.0f;
        const Strided<D> qs(p.q.p + row_at(p, p.q, w, 0), p.q.l, p.R), gs(p.go.p + row_at(p, p.go, w, 0), p.go.l, p.R);
        auto request = [&](uint32_t blk, float *to) {
            if (p.strided) {
                qs.template stage<RB, DMA>(to, (int)blk * RB);
                gs.template stage<RB, DMA>(to + RB * D, (int)blk * RB);
            } else {
                auto at = [&](int r) { return min(blk * RB + r, (uint32_t)p.R - 1); };
                stage<D, RB, DMA>(to, [&](int r) { return p.q.p + row_at(p, p.q, w, at(r)); });
                stage<D, RB, DMA>(to + RB * D, [&](int r) { return p.go.p + row_at(p, p.go, w, at(r)); });
            }
            if (tid < RB) {
                const uint32_t r = blk * RB + tid;
                lreg = r < (uint32_t)p.R ? p.lse[(int64_t)w.pair * p.R + r] : inf;  // a row past the end: every exponential is 0
                dreg = r < (uint32_t)p.R ? p.delta[(int64_t)w.pair * p.R + r] : 0.0f;
            }
        };
        uint32_t first, last;
        split_range((p.R + RB - 1) / RB, w.split, p.splits, &first, &last);
        // a wavefront none of whose keys is visible only helps to stage
        const bool works = __builtin_amdgcn_ballot_w64(seen) != 0;
        auto step = [&](uint32_t blk, float *tile, float *rows, float *other) {
            if (tid < RB) { rows[tid] = lreg * LOG2E; rows[RB + tid] = dreg; }
            arrived();
            __syncthreads();
            if (blk + 1 < last) request(blk + 1, other);
            if (!works) return;
            __builtin_amdgcn_sched_barrier(0);  // the parts one after the other: all operands at once do not fit the registers
            const float *qt = tile + rw * D, *gt = tile + (RB + rw) * D, *ls = rows + rw, *dl = rows + RB + rw;
            floatx16 s = scores<D>(qt, k, c, h);
            __builtin_amdgcn_sched_barrier(0);
            floatx16 dp = scores<D>(gt, v, c, h);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 l4 = *reinterpret_cast<const f32x4 *>(&ls[8 * g + 4 * h]), d4 = *reinterpret_cast<const f32x4 *>(&dl[8 * g + 4 * h]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[4 * g + i] - l4[i]);
                    s[4 * g + i] = e;
                    dp[4 * g + i] = e * (dp[4 * g + i] - d4[i]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            accumulate<D>(gt, s, gv, c, h);
            __builtin_amdgcn_sched_barrier(0);
            accumulate<D>(qt, dp, gk, c, h);
        };
        if (first < last) request(first, lds0);
        k.scale(p.scale * LOG2E);
        for (uint32_t blk = first; blk < last; blk += 2) {
            step(blk, lds0, rows0, lds1);
            if (blk + 1 < last) step(blk + 1, lds1, rows1, lds0);
        }
    }
    const bool writes = merge_waves<CW, SLOT>(lds0, wave, lane, [&](float *to) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) { to[16 * d + i] = gk[d][i]; to[16 * (ND + d) + i] = gv[d][i]; }
    }, [&](const float *from) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) { gk[d][i] += from[16 * d + i]; gv[d][i] += from[16 * (ND + d) + i]; }
    });
    if (!writes || j >= p.Lk) return;
    if (!seen) {
#pragma unroll
        for (int d = 0; d < ND; ++d) gk[d] = gv[d] = zero16();
    }
    if (p.splits > 1) {
        const int64_t at = (((int64_t)w.split * p.pairs + w.pair) * p.Lk + j) * D;
        write_column<D>(p.part_k + at, gk, p.scale, h);
        write_column<D>(p.part_v + at, gv, 1.0f, h);
    } else {
        write_column<D>(const_cast<float *>(p.gk.p) + w.b * p.gk.b + w.g * p.gk.h + (int64_t)j * p.gk.l, gk, p.scale, h);
        write_column<D>(const_cast<float *>(p.gv.p) + w.b * p.gv.b + w.g * p.gv.h + (int64_t)j * p.gv.l, gv, 1.0f, h);
    }
}

template <int D, int CW, bool DMA>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 32 ? 3 : 2))) cross_gkv_kernel(const CrossP p) {
    __shared__ __attribute__((aligned(16))) float lds0[256 / CW * D], lds1[256 / CW * D];  // two buffers of rows of Q and dO
    __shared__ __attribute__((aligned(16))) float rows0[256 / CW], rows1[256 / CW];
    __shared__ int lds_end[8];
    gkv_work<D, CW, DMA>(p, blockIdx.x, lds0, lds1, rows0, rows1, lds_end);
}

// ---- both gradients in one launch, where each on its own leaves compute units idle at its end: the first key_ids workgroups
// (a multiple of 8) take keys, the others rows.  All launches of a gradient, apart and together: 7 x 2 key heads of 1332 rows, 1001
// to 501 keys of size 32 91 and 80 us; 12 heads of 512 x 512, size 64, 8 sequences 247 and 223 us, 16 408 and 432 us, with lengths
// 512 to 272 8 sequences 217 and 185 us, 16 364 and 351 us, 32 661 and 676 us.
template <int D, bool DMA>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D == 32 ? 3 : 2))) cross_both_kernel(const CrossP keys, const CrossP rows, uint32_t key_ids) {
    __shared__ __attribute__((aligned(16))) float lds0[128 * D], lds1[128 * D];
    __shared__ __attribute__((aligned(16))) float rows0[128], rows1[128];
    __shared__ int lds_end[8];
    if (blockIdx.x >= key_ids) gq_work<D, 2, DMA, true>(rows, blockIdx.x - key_ids, lds0, lds1, lds_end);
    else if (keys.ends || blockIdx.x < keys.tiles * keys.pairs * keys.splits) gkv_work<D, 2, DMA>(keys, blockIdx.x, lds0, lds1, rows0, rows1, lds_end);
}

// In front of it: the lengths (the first `ends` workgroups), and delta by D / 4 lanes a row.
template <int D>
__global__ void __launch_bounds__(256) cross_front_kernel(const CrossP p, uint32_t ends) {
    __shared__ int lds[4];
    if (blockIdx.x < ends) {
        const int end = visible_end(p, blockIdx.x, lds);
        if (threadIdx.x == 0) p.ends[blockIdx.x] = end;
        return;
    }
    constexpr int LPR = D / 4;
    const uint32_t total = p.pairs * p.R, row = (blockIdx.x - ends) * (256 / LPR) + threadIdx.x / LPR, at = min(row, total - 1);
    Work w;
    w.pair = at / p.R;
    w.b = (int)fdiv(w.pair, p.d_g);
    w.g = (int)w.pair - w.b * p.G;
    const uint32_t r = at - w.pair * p.R, col = threadIdx.x % LPR * 4;
    const f32x4 o = load4(p.o.p + row_at(p, p.o, w, r) + col), g = load4(p.go.p + row_at(p, p.go, w, r) + col);
    const float sum = group_sum<D>(__builtin_fmaf(o.w, g.w, __builtin_fmaf(o.z, g.z, __builtin_fmaf(o.y, g.y, o.x * g.x))));
    if (row < total && col == 0) p.delta[row] = sum;
}

// out[row] = sum of the splits' rows, in order: D / 4 lanes a row.  Rows are [batch][heads][length].  The gradients that were
// split, one after the other in one launch.
struct SumJob {
    const float *part;
    Rows out;
    uint32_t total, splits, heads, length;
    uint32_t first_block;
};
struct SumJobs {
    SumJob job[3];
    int count;
};
template <int D>
__global__ void __launch_bounds__(256) cross_sum_kernel(const SumJobs jobs) {
    constexpr int LPR = D / 4;
    int which = 0;
    while (which + 1 < jobs.count && blockIdx.x >= jobs.job[which + 1].first_block) ++which;
    const SumJob &j = jobs.job[which];
    const uint32_t row = (blockIdx.x - j.first_block) * (256 / LPR) + threadIdx.x / LPR, col = threadIdx.x % LPR * 4;
    if (row >= j.total) return;
    f32x4 acc = *reinterpret_cast<const f32x4 *>(j.part + (int64_t)row * D + col);
    for (uint32_t i = 1; i < j.splits; ++i) acc += *reinterpret_cast<const f32x4 *>(j.part + ((int64_t)i * j.total + row) * D + col);
    const uint32_t bh = row / j.length;
    store4(const_cast<float *>(j.out.p) + bh / j.heads * j.out.b + bh % j.heads * j.out.h + (int64_t)(row - bh * j.length) * j.out.l + col, acc);
}

int check_operand(sg_ctx *ctx, const sg_tensor *t, int64_t n, int64_t heads, int64_t len, int64_t D, const char *who, Rows *r) {
    const int rc = sg_check_f32(ctx, t, who);
    if (rc != SG_OK) return rc;
    if (t->rank != 4) return sg_fail(ctx, SG_ERR_SHAPE, "%s: rank %d, expected [batch, heads, length, head size]", who, t->rank);
    if (t->extents[0] != n || t->extents[1] != heads || t->extents[2] != len || t->extents[3] != D)
        return sg_fail(ctx, SG_ERR_SHAPE, "%s: [%lld, %lld, %lld, %lld], expected [%lld, %lld, %lld, %lld]", who, (long long)t->extents[0], (long long)t->extents[1],
                       (long long)t->extents[2], (long long)t->extents[3], (long long)n, (long long)heads, (long long)len, (long long)D);
    if (t->strides[3] != 1) return sg_fail(ctx, SG_ERR_SHAPE, "%s: the head dimension must have unit stride", who);
    *r = {(const float *)t->base + t->offset, t->strides[0], t->strides[1], t->strides[2]};
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
    // A launch has fewer than 2^32 threads, in workgroups of 256, rounded up to the 8 XCDs.  (More than one tile of rows or keys a
    // pair leaves room: 2^31 elements are the most of an operand.)
    if (N * G > (1 << 24) - 8) return sg_fail(ctx, SG_ERR_SHAPE, "cross attention: %lld sequences of %lld key heads (2^24 - 8 together at most)", (long long)N, (long long)G);
    if ((rc = check_operand(ctx, q, N, H, Lq, D, "cross attention q", &p.q)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, k, N, G, Lk, D, "cross attention k", &p.k)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, v, N, G, Lk, D, "cross attention v", &p.v)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, out, N, H, Lq, D, "cross attention out", &p.o)) != SG_OK) return rc;
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
    p.R = (int)(H / G * Lq);
    p.pairs = (uint32_t)(N * G);
    p.d_lq = sg_make_fastdiv((uint32_t)Lq);
    p.d_g = sg_make_fastdiv((uint32_t)G);
    p.d_pairs = sg_make_fastdiv(p.pairs);
    return SG_OK;
}

// 16-byte aligned rows less than 16 MB apart: loads straight into LDS take them.
bool aligned_rows(const Rows &r) { return ((uintptr_t)r.p) % 16 == 0 && r.b % 4 == 0 && r.h % 4 == 0 && r.l % 4 == 0 && r.l < (1 << 22); }

// How a kernel takes an axis of `own` rows (or keys) that walk `other` of the other side: wavefronts of a workgroup side by
// side on it (the 4 / waves others share the blocks of the walk), and workgroups a walk is split over.
struct Plan {
    int waves;
    uint32_t splits;
};

// The plan of the least estimated time: what the busiest compute unit has of workgroups, each so many blocks of `step_us` and
// 1.5 us to begin and end, at three quarters of the rate where only one is there to work; a join of 4 us and 0.4 a split; a
// fifth more for the blocks that smaller tiles load more often.  With a mask, of which only the device knows the lengths,
// three quarters of the keys are taken to be visible: finer workgroups then level what the lengths leave uneven.
// (1332 rows of 14 pairs, 1001 keys of size 32, lengths 1001 to 501: forward 4 wavefronts side by side in 3 splits 33 us and a
// join of 5, 1 wavefront 29 and none; gradient of the queries 43 and a sum, 39 and none.  512 rows of 384 pairs, 512 keys of
// size 64: 4 wavefronts 186 and 266 us, 2 wavefronts 220 and 300.)
Plan plan(const sg_ctx *ctx, const CrossP &p, int64_t D, int own, int other, int least_waves, int most_waves, double step_us) {
    const uint64_t cus = (uint64_t)(ctx->num_cus > 0 ? ctx->num_cus : 256);
    Plan best = {most_waves, 1};
    double least = 1e30;
    for (int w = most_waves; w >= least_waves; w /= 2) {
        const uint64_t units = (uint64_t)((own + 32 * w - 1) / (32 * w)) * p.pairs;
        const uint32_t blocks = (uint32_t)((other + 128 / w - 1) / (128 / w));
        for (uint32_t s = 1; s <= 64 && (s == 1 || (s <= blocks / 2 && units * s <= 3 * cus)); ++s) {
            const uint64_t most = ((p.mask ? units * s * 3 / 4 : units * s) + cus - 1) / cus;
            const bool alone = most == 1 || (D == 64 && w == 1);  // 128 KB of LDS
            const double block_us = step_us * (alone ? 1.33 : 1.0) * (w == 4 ? 1.0 : w == 2 ? 1.15 : 1.2);
            const double cost = (double)most * ((blocks + s - 1) / s * block_us + 1.5) + (s > 1 ? 4.0 + 0.4 * s : 0.0);
            if (cost < least) { least = cost; best = {w, s}; }
        }
    }
    return best;
}

void set_tiles(CrossP &p, uint32_t tiles, uint32_t splits) {
    p.tiles = tiles;
    p.splits = splits;
    p.spread = (uint64_t)p.pairs * splits < 64;  // an XCD would have fewer than 8 units, of different lengths
    p.d_tiles = sg_make_fastdiv(p.tiles);
}

// Lengths in front of the launches, where there are more workgroups than `each` for a compute unit and lengths to order them by.
bool orders_lengths(const sg_ctx *ctx, const CrossP &p, uint64_t workgroups, uint32_t each) {
    return p.mask && p.N > 1 && p.N <= 256 && workgroups > each * (uint64_t)(ctx->num_cus > 0 ? ctx->num_cus : 256);
}

}  // namespace

#define SG_CROSS_ROWS_(KERNEL, D_, RW, DMA, GRID)                                                                       \
    do {                                                                                                                \
        if (RW == 4) hipLaunchKernelGGL((KERNEL<D_, 4, DMA>), GRID, dim3(256), 0, ctx->stream, p);                      \
        else if (RW == 2) hipLaunchKernelGGL((KERNEL<D_, 2, DMA>), GRID, dim3(256), 0, ctx->stream, p);                 \
        else hipLaunchKernelGGL((KERNEL<D_, 1, DMA>), GRID, dim3(256), 0, ctx->stream, p);                              \
    } while (0)
#define SG_CROSS_ROWS(KERNEL, RW, DMA, GRID)                                                                            \
    do {                                                                                                                \
        if (D == 64 && DMA) SG_CROSS_ROWS_(KERNEL, 64, RW, true, GRID);                                                 \
        else if (D == 64) SG_CROSS_ROWS_(KERNEL, 64, RW, false, GRID);                                                  \
        else if (DMA) SG_CROSS_ROWS_(KERNEL, 32, RW, true, GRID);                                                       \
        else SG_CROSS_ROWS_(KERNEL, 32, RW, false, GRID);                                                               \
    } while (0)

extern "C" int sg_cross_attention(sg_ctx *ctx, const sg_tensor *q, const sg_tensor *k, const sg_tensor *v, const sg_tensor *mask, float scale,
                                  const sg_tensor *out, const sg_tensor *lse) {
    CrossP p{};
    int rc = check_call(ctx, q, k, v, mask, out, lse, true, p);
    if (rc != SG_OK) return rc;
    if (!ctx) return SG_ERR_ARG;
    p.scale = scale;
    sg_device_guard guard(ctx);
    const int64_t D = q->extents[3];
    const bool few = p.R <= 8;
    const uint32_t total = p.pairs * (uint32_t)p.R;
    Plan how;
    if (few) {
        // Bound by memory: two workgroups for each compute unit, of 128 keys at least.  From as many pairs as compute units on
        // nothing is split: the join's launch costs more than it levels.
        const uint32_t cus = (uint32_t)(ctx->num_cus > 0 ? ctx->num_cus : 256), most = (uint32_t)p.Lk / 128;
        how.splits = p.pairs >= cus ? 1 : (2 * cus + p.pairs - 1) / p.pairs;
        how.splits = how.splits > most ? most : how.splits;
        how.splits = how.splits < 1 ? 1 : how.splits > 64 ? 64 : how.splits;
        how.waves = 1;
    } else {
        how = plan(ctx, p, D, p.R, p.Lk, 1, 4, D == 64 ? 1.7 : 1.1);
    }
    const int rw = how.waves;
    const uint32_t tiles = few ? 1 : (uint32_t)((p.R + 32 * rw - 1) / (32 * rw));
    set_tiles(p, tiles, how.splits);
    sg_workspace space(ctx);
    if (p.splits > 1) {
        if ((rc = space.take((uint64_t)p.splits * total * (D + 2) * 4)) != SG_OK) return rc;
        p.part_o = (float *)space.p;
        p.part_ml = p.part_o + (uint64_t)p.splits * total * D;
    } else if (!few && orders_lengths(ctx, p, (uint64_t)tiles * p.pairs, 2)) {
        if ((rc = space.take((uint64_t)p.N * 4)) != SG_OK) return rc;
        p.ends = (int *)space.p;
        hipLaunchKernelGGL(cross_ends_kernel, dim3((unsigned)p.N), dim3(256), 0, ctx->stream, p);
        SG_CHECK_LAUNCH(ctx, "cross_attention lengths");
    }
    const dim3 grid(p.tiles * p.pairs * p.splits);
#define SG_CROSS_FEW(D_, ROWS, UNROLL) hipLaunchKernelGGL((cross_few_kernel<D_, ROWS, UNROLL>), grid, dim3(256), 0, ctx->stream, p)
    const bool dma = aligned_rows(p.q) && aligned_rows(p.k) && aligned_rows(p.v);
    if (!few) SG_CROSS_ROWS(cross_forward_kernel, rw, dma, grid);
    else if (D == 64) {
        if (p.R == 1) SG_CROSS_FEW(64, 1, 8);
        else if (p.R == 2) SG_CROSS_FEW(64, 2, 8);
        else if (p.R <= 4) SG_CROSS_FEW(64, 4, 4);
        else SG_CROSS_FEW(64, 8, 4);
    } else {
        if (p.R == 1) SG_CROSS_FEW(32, 1, 4);
        else if (p.R == 2) SG_CROSS_FEW(32, 2, 4);
        else if (p.R <= 4) SG_CROSS_FEW(32, 4, 4);
        else SG_CROSS_FEW(32, 8, 4);
    }
#undef SG_CROSS_FEW
    SG_CHECK_LAUNCH(ctx, "cross_attention");
    if (p.splits > 1) {
        const dim3 rows((unsigned)((total + 1024 / D - 1) / (1024 / D)));
        if (D == 64) hipLaunchKernelGGL((cross_join_kernel<64>), rows, dim3(256), 0, ctx->stream, p);
        else hipLaunchKernelGGL((cross_join_kernel<32>), rows, dim3(256), 0, ctx->stream, p);
        SG_CHECK_LAUNCH(ctx, "cross_attention join");
    }
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
    if ((rc = check_operand(ctx, gout, N, p.H, p.Lq, D, "sg_cross_attention_grad gout", &p.go)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, gq, N, p.H, p.Lq, D, "sg_cross_attention_grad gq", &p.gq)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, gk, N, p.G, p.Lk, D, "sg_cross_attention_grad gk", &p.gk)) != SG_OK) return rc;
    if ((rc = check_operand(ctx, gv, N, p.G, p.Lk, D, "sg_cross_attention_grad gv", &p.gv)) != SG_OK) return rc;
    if ((rc = check_apart(ctx, gq, "sg_cross_attention_grad gq")) != SG_OK) return rc;
    if ((rc = check_apart(ctx, gk, "sg_cross_attention_grad gk")) != SG_OK) return rc;
    if ((rc = check_apart(ctx, gv, "sg_cross_attention_grad gv")) != SG_OK) return rc;
    if (!ctx) return SG_ERR_ARG;
    p.scale = scale;
    p.strided = p.H == p.G || (p.q.h == p.Lq * p.q.l && p.go.h == p.Lq * p.go.l);
    sg_device_guard guard(ctx);
    const uint64_t total = (uint64_t)p.pairs * p.R, keys = (uint64_t)p.pairs * p.Lk;
    const bool dma = aligned_rows(p.q) && aligned_rows(p.k) && aligned_rows(p.v) && aligned_rows(p.o) && aligned_rows(p.go);
    // One launch for both gradients, while their workgroups of 64 rows or keys are few enough for a launch's end to count (8 for a
    // compute unit, 12 where lengths differ), and O and dO, of which delta has to be made in front then, are 64 MB at most.
    const uint64_t tiles64 = (uint64_t)((p.R + 63) / 64 + (p.Lk + 63) / 64) * p.pairs, cus = (uint64_t)(ctx->num_cus > 0 ? ctx->num_cus : 256);
    const bool both = p.R > 32 && total * D * 8 <= (64u << 20) && tiles64 <= (p.mask ? 12 : 8) * cus;
    const Plan by_rows = plan(ctx, p, D, p.R, p.Lk, both ? 2 : 1, both ? 2 : 4, D == 64 ? 2.6 : 1.6);
    // 128 keys a workgroup only where all are visible: smaller tiles waste less of a sequence's last one and level better
    // (32 x 12 heads of 512 x 512: 446 us against 473 with 64 keys; with lengths 512 to 272: 423 against 404 us); and up to 32
    // rows, all of which a wavefront takes (15 rows, 14 x 8 heads, 4048 keys of size 32: 99 us with 64 keys, 53 us).
    const Plan by_keys = plan(ctx, p, D, p.Lk, p.R, p.R <= 32 ? 4 : 2, both || (p.mask && p.R > 32) ? 2 : 4, D == 64 ? 3.4 : 2.0);
    const int rw = by_rows.waves, cw = by_keys.waves;
    const uint32_t row_tiles = (uint32_t)((p.R + 32 * rw - 1) / (32 * rw)), key_tiles = (uint32_t)((p.Lk + 32 * cw - 1) / (32 * cw));
    const uint32_t row_splits = by_rows.splits, key_splits = by_keys.splits;
    // delta and the lengths, the split sums of both kernels
    const uint64_t rows_part = row_splits > 1 ? row_splits * total * D : 0, keys_part = key_splits > 1 ? 2 * key_splits * keys * D : 0;
    const uint64_t delta_floats = (total + (uint64_t)p.N + 3) / 4 * 4;
    sg_workspace space(ctx);
    if ((rc = space.take((delta_floats + rows_part + keys_part) * 4)) != SG_OK) return rc;
    p.delta = (float *)space.p;
    p.part_o = p.delta + delta_floats;
    p.part_k = p.part_o + rows_part;
    p.part_v = p.part_k + key_splits * keys * D;
    if (both) {
        const uint32_t ends = p.mask && p.N <= 256 ? (uint32_t)p.N : 0;
        if (ends) p.ends = (int *)(p.delta + total);
        const dim3 front(ends + (unsigned)((total + 1024 / D - 1) / (1024 / D)));
        if (D == 64) hipLaunchKernelGGL((cross_front_kernel<64>), front, dim3(256), 0, ctx->stream, p, ends);
        else hipLaunchKernelGGL((cross_front_kernel<32>), front, dim3(256), 0, ctx->stream, p, ends);
        SG_CHECK_LAUNCH(ctx, "cross_attention_grad delta");
        CrossP rows = p;
        set_tiles(rows, row_tiles, row_splits);
        set_tiles(p, key_tiles, key_splits);
        const uint32_t key_ids = (p.tiles * p.pairs * p.splits + 7) / 8 * 8;
        const dim3 grid(key_ids + rows.tiles * rows.pairs * rows.splits);
        if (D == 64 && dma) hipLaunchKernelGGL((cross_both_kernel<64, true>), grid, dim3(256), 0, ctx->stream, p, rows, key_ids);
        else if (D == 64) hipLaunchKernelGGL((cross_both_kernel<64, false>), grid, dim3(256), 0, ctx->stream, p, rows, key_ids);
        else if (dma) hipLaunchKernelGGL((cross_both_kernel<32, true>), grid, dim3(256), 0, ctx->stream, p, rows, key_ids);
        else hipLaunchKernelGGL((cross_both_kernel<32, false>), grid, dim3(256), 0, ctx->stream, p, rows, key_ids);
        SG_CHECK_LAUNCH(ctx, "cross_attention_grad");
    } else {
        if (orders_lengths(ctx, p, (uint64_t)key_tiles * key_splits * p.pairs, 1)) {
            p.ends = (int *)(p.delta + total);
            hipLaunchKernelGGL(cross_ends_kernel, dim3((unsigned)p.N), dim3(256), 0, ctx->stream, p);
            SG_CHECK_LAUNCH(ctx, "cross_attention_grad lengths");
        }
        set_tiles(p, row_tiles, row_splits);
        SG_CROSS_ROWS(cross_gq_kernel, rw, dma, dim3(p.tiles * p.pairs * p.splits));
        SG_CHECK_LAUNCH(ctx, "cross_attention_grad queries");
        set_tiles(p, key_tiles, key_splits);
        uint32_t workgroups = p.tiles * p.pairs * p.splits;
        if (p.ends) workgroups = (workgroups + 7) / 8 * 8;
        const dim3 grid(workgroups);
#define SG_CROSS_KEYS(D_, CW, DMA) hipLaunchKernelGGL((cross_gkv_kernel<D_, CW, DMA>), grid, dim3(256), 0, ctx->stream, p)
#define SG_CROSS_KEYS_(D_, CW)                 \
        do {                                       \
            if (dma) SG_CROSS_KEYS(D_, CW, true);  \
            else SG_CROSS_KEYS(D_, CW, false);     \
        } while (0)
        if (D == 64 && cw == 4) SG_CROSS_KEYS_(64, 4);
        else if (D == 64) SG_CROSS_KEYS_(64, 2);
        else if (cw == 4) SG_CROSS_KEYS_(32, 4);
        else SG_CROSS_KEYS_(32, 2);
#undef SG_CROSS_KEYS_
#undef SG_CROSS_KEYS
        SG_CHECK_LAUNCH(ctx, "cross_attention_grad keys and values");
    }
    SumJobs sums{};
    uint32_t blocks = 0;
    auto add = [&](const float *part, const Rows &out, uint64_t rows, uint32_t splits, int heads, int length) {
        if (splits == 1) return;
        sums.job[sums.count++] = {part, out, (uint32_t)rows, splits, (uint32_t)heads, (uint32_t)length, blocks};
        blocks += (uint32_t)((rows + 1024 / D - 1) / (1024 / D));
    };
    add(p.part_o, p.gq, total, row_splits, p.H, p.Lq);
    add(p.part_k, p.gk, keys, key_splits, p.G, p.Lk);
    add(p.part_v, p.gv, keys, key_splits, p.G, p.Lk);
    if (blocks) {
        if (D == 64) hipLaunchKernelGGL((cross_sum_kernel<64>), dim3(blocks), dim3(256), 0, ctx->stream, sums);
        else hipLaunchKernelGGL((cross_sum_kernel<32>), dim3(blocks), dim3(256), 0, ctx->stream, sums);
        SG_CHECK_LAUNCH(ctx, "cross_attention_grad sums");
    }
    return SG_OK;
}
