// Embedding lookup with scaling and its gradient for gfx950.
//   forward:  out[i, :] = scale * table[id_i, :]            (zeros where id_i is no row of the table)
//   backward: gtable[v, :] = scale * sum_{i: id_i = v} gout[i, :]
// Both are bound by memory: a row is read once and written once.
#include "rows.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // 16 bytes at any element

// Columns c .. c + 3 of a row of E.  Where fewer than 4 are left the row's last 4 are taken instead: two lanes then do the
// same for some columns and store the same values there, but no load waits behind a branch (a row of any width begins
// anywhere; 21969 tokens of 145: lookup 7.5, sums of the gradient 10.9, join 7.8 us, with 4 bytes a load 9.8, 13.5 and 9.6).
// NARROW: E below 4.  NT: past the caches.
template <bool NARROW, bool NT = false>
__device__ __forceinline__ f32x4 load_cols(const float *row, uint32_t c, uint32_t E) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (NARROW) {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (c + j < E) v[j] = row[c + j];
    } else if (c < E) {
        const f32x4_any *p = reinterpret_cast<const f32x4_any *>(row + min(c, E - 4));
        v = NT ? __builtin_nontemporal_load(p) : *p;
    }
    return v;
}
template <bool NARROW, bool NT = false>
__device__ __forceinline__ void store_cols(float *row, uint32_t c, uint32_t E, f32x4 v) {
    if (NARROW) {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (c + j < E) row[c + j] = v[j];
    } else if (c < E) {
        f32x4_any *p = reinterpret_cast<f32x4_any *>(row + min(c, E - 4));
        if (NT) __builtin_nontemporal_store(v, p);
        else *p = v;
    }
}

struct EmbP {
    const float *table;
    const uint32_t *ids;
    float *out;
    sg_rows id_rows;
    uint32_t n, E, V, pieces;
    int64_t table_stride;
    float scale;
};

// A wavefront writes 256 columns of one token's row, 16 bytes a lane: every piece of every row is a wavefront of its
// own, so that the few rows of a serving batch are in flight together too.  Rows of 768: 8 tokens 2.6 us, the time of a launch;
// 4096 tokens 6.4 us (25 MB, 3.9 TB/s); 32768 tokens, three tenths of them none, 20 us (101 MB written past the caches, 5 TB/s).
template <bool NARROW, bool NT>
__global__ void __launch_bounds__(256) embedding_kernel(const EmbP p) {
    const uint64_t unit = (uint64_t)sg_workgroup() * 4 + (threadIdx.x >> 6);
    if (unit >= (uint64_t)p.n * p.pieces) return;
    const uint32_t token = (uint32_t)(unit / p.pieces), piece = (uint32_t)(unit - (uint64_t)token * p.pieces);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t id = p.ids[sg_row_offset(p.id_rows, token)];
    const bool known = id < p.V;
    const float *src = p.table + (known ? (int64_t)id * p.table_stride : 0);
    float *dst = p.out + (int64_t)token * p.E;
    const uint32_t c = piece * 256 + lane * 4;
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (known) v = load_cols<NARROW>(src, c, p.E) * p.scale;
    store_cols<NARROW, NT>(dst, c, p.E, v);
}

// ---- gradient.  The tokens are sorted by id (stable, so a row's tokens stay in order), unknown ones behind the last row;
// the sorted list is cut into chunks, each summed by wavefronts of its own; runs of one id that cross chunks leave partial
// sums, which a last launch joins.  The order of every sum follows from the ids alone.
//
// Bound by memory: the gradient table is written once (rows without tokens are most of it) and gout read once.  The table
// is cleared by the workgroups that ride in the sorting launches, which are otherwise a few workgroups on an idle chip;
// rows with tokens are written a second time by the sums.  Table of 30522 x 768 (94 MB, 14 us at the rate of a fill): 4096
// tokens 29 us, of which 17.6 are the sort beside the clearing, 7.4 the sums, 4.0 the join; 32768 tokens 52 us: count 6.5, two
// moves of 9.8, sums 19 (71 MB of gout, 3.7 TB/s), join 6.7.
constexpr int SORT_THREADS = 1024, SORT_WAVES = SORT_THREADS / 64;
constexpr uint32_t MAX_DIGITS = 512;       // 9 bits a pass: two passes up to 262143 rows
constexpr uint32_t SINGLE = SORT_THREADS * 8;  // tokens that one workgroup sorts in LDS in one launch
constexpr uint32_t FILL = 8;               // 16-byte pieces a thread of a clearing workgroup writes

struct SortP {
    const uint32_t *ids;       // first pass: the ids themselves
    const uint32_t *key_in, *pos_in;
    uint32_t *key_out, *pos_out;
    uint32_t *hist, *next_hist;  // [tile][digit] of this pass; of the next one, if this one counts it
    sg_rows id_rows;
    uint32_t n, V, tiles, shift, digits, from_ids;
    uint32_t bits, passes;     // of the single-workgroup form
    float *fill;               // what this launch clears
    uint64_t fill_floats;
    uint32_t fill_vec;
};

__device__ __forceinline__ void clear_part(const SortP &p, uint32_t block) {
    const uint64_t base = (uint64_t)block * (SORT_THREADS * FILL * 4);
#pragma unroll
    for (uint32_t k = 0; k < FILL; ++k) {
        const uint64_t i = base + ((uint64_t)k * SORT_THREADS + threadIdx.x) * 4;
        if (i >= p.fill_floats) return;
        if (p.fill_vec && i + 4 <= p.fill_floats) __builtin_nontemporal_store(f32x4{0.0f, 0.0f, 0.0f, 0.0f}, reinterpret_cast<f32x4 *>(p.fill + i));
        else for (uint64_t j = i; j < i + 4 && j < p.fill_floats; ++j) p.fill[j] = 0.0f;
    }
}

// Item k of a thread is token first + (wave * ITEMS + k) * 64 + lane: a wavefront's tokens are consecutive.
__device__ __forceinline__ uint32_t item_index(uint32_t items, uint32_t k) { return ((threadIdx.x >> 6) * items + k) * 64 + (threadIdx.x & 63); }

__device__ __forceinline__ uint32_t key_of(const SortP &p, uint32_t i) {
    const uint32_t id = p.ids[sg_row_offset(p.id_rows, i)];
    return id < p.V ? id : p.V;
}

// rank[k]: tokens of the same digit in front of item k in this tile, for the first `items` of ITEMS registers.  counts:
// [wave][digit], zeroed, in LDS; left as the exclusive sums over the wavefronts, with the tile's counts in totals.  Items
// that are not there have digit `digits`, which nothing counts.
template <uint32_t ITEMS>
__device__ __forceinline__ void rank_items(const uint32_t *digit, uint32_t *rank, uint16_t *counts, uint32_t *totals, uint32_t digits, uint32_t items) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t below = (1ull << lane) - 1;
    volatile uint16_t *mine = counts + wave * digits;
    uint32_t low[ITEMS], high[ITEMS];  // lanes whose digit differs; all items bit by bit, each alone would wait for its own ballots
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) low[k] = high[k] = 0;
    for (uint32_t bit = 1; bit < digits; bit <<= 1)
#pragma unroll
        for (uint32_t k = 0; k < ITEMS; ++k) {
            const bool set = (digit[k] & bit) != 0;
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(set);
            const uint32_t all = set ? ~0u : 0u;
            low[k] |= (uint32_t)lanes ^ all;
            high[k] |= (uint32_t)(lanes >> 32) ^ all;
        }
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        if (k >= items) break;
        const uint64_t same = __builtin_amdgcn_ballot_w64(digit[k] < digits) & ~((uint64_t)high[k] << 32 | low[k]);
        rank[k] = 0;
        if (digit[k] < digits) {
            const uint32_t before = mine[digit[k]];
            __builtin_amdgcn_wave_barrier();  // every lane has read before the first of its digit writes
            rank[k] = before + (uint32_t)__popcll(same & below);
            if ((same & below) == 0) mine[digit[k]] = (uint16_t)(before + (uint32_t)__popcll(same));
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    if (threadIdx.x < digits) {
        uint32_t x[SORT_WAVES], sum = 0;
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) x[w] = counts[w * digits + threadIdx.x];
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            counts[w * digits + threadIdx.x] = (uint16_t)sum;  // below the tile's 8192
            sum += x[w];
        }
        totals[threadIdx.x] = sum;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k)
        if (k < items && digit[k] < digits) rank[k] += counts[wave * digits + digit[k]];
}

// Exclusive prefix sums of totals[0..digits) in LDS, in place.  scratch: one word per wavefront.
__device__ __forceinline__ void prefix_digits(uint32_t *totals, uint32_t *scratch, uint32_t digits) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t x = threadIdx.x < digits ? totals[threadIdx.x] : 0;
    uint32_t sum = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = (uint32_t)__shfl_up((int)sum, o, 64);
        if ((int)lane >= o) sum += y;
    }
    if (lane == 63) scratch[wave] = sum;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < MAX_DIGITS / 64; ++w)
        if (w < wave) sum += scratch[w];
    if (threadIdx.x < digits) totals[threadIdx.x] = sum - x;
    __syncthreads();
}

// Up to 8192 tokens: workgroup 0 sorts them, all passes in LDS; the others clear the table.  (Up to 4096 tokens in half the
// registers and LDS, so that two clearing workgroups share a compute unit.)  Two passes: 327 tokens 5.6 us, 3559 tokens in one pass
// 6.7, 7363 tokens 17.6.
template <uint32_t ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) embedding_sort_kernel(const SortP p) {
    __shared__ uint32_t keys[SORT_THREADS * ITEMS], totals[MAX_DIGITS], scratch[SORT_WAVES];
    __shared__ uint16_t places[SORT_THREADS * ITEMS], counts[SORT_WAVES * MAX_DIGITS];
    if (blockIdx.x > 0) {
        clear_part(p, blockIdx.x - 1);
        return;
    }
    uint32_t key[ITEMS], pos[ITEMS], digit[ITEMS], rank[ITEMS];
    const uint32_t items = (p.n + SORT_THREADS - 1) / SORT_THREADS;  // per thread; the rest of the registers stay empty
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        const uint32_t i = item_index(items, k);
        pos[k] = i;
        key[k] = k < items && i < p.n ? key_of(p, i) : 0;
    }
    for (uint32_t pass = 0; pass < p.passes; ++pass) {
        const uint32_t shift = pass * p.bits, digits = 1u << p.bits;
        for (uint32_t i = threadIdx.x; i < SORT_WAVES * digits; i += SORT_THREADS) counts[i] = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < ITEMS; ++k) {
            const bool there = k < items && item_index(items, k) < p.n;
            digit[k] = there ? (key[k] >> shift) & (digits - 1) : digits;
        }
        rank_items<ITEMS>(digit, rank, counts, totals, digits, items);
        prefix_digits(totals, scratch, digits);
#pragma unroll
        for (uint32_t k = 0; k < ITEMS; ++k)
            if (digit[k] < digits) {
                const uint32_t to = totals[digit[k]] + rank[k];
                keys[to] = key[k];
                places[to] = (uint16_t)pos[k];
            }
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < ITEMS; ++k) {
            const uint32_t i = item_index(items, k);
            if (k < items && i < p.n) { key[k] = keys[i]; pos[k] = places[i]; }
        }
        __syncthreads();
    }
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        const uint32_t i = item_index(items, k);
        if (k < items && i < p.n) { p.key_out[i] = key[k]; p.pos_out[i] = pos[k]; }
    }
}

// More tokens: a launch counts every tile's digits, the next moves every token to its place of this pass, and counts the
// next pass's digits where the tokens land, in LDS first, if the tiles' counts fit there (else a launch of its own does).
// Tiles of ITEMS tokens a thread: 2 up to 131072 tokens (32768 tokens: a move 9.8 us, with 4 11.9, with 1 9.6), then 4, since
// every tile adds up the counts of all.
constexpr uint32_t NEXT_COUNTS = 8192;
template <uint32_t ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) embedding_count_kernel(const SortP p) {
    __shared__ uint32_t count[MAX_DIGITS];
    if (blockIdx.x >= p.tiles) {
        clear_part(p, blockIdx.x - p.tiles);
        return;
    }
    if (threadIdx.x < p.digits) count[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        const uint32_t i = blockIdx.x * (SORT_THREADS * ITEMS) + k * SORT_THREADS + threadIdx.x;
        if (i < p.n) atomicAdd(&count[((p.from_ids ? key_of(p, i) : p.key_in[i]) >> p.shift) & (p.digits - 1)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < p.digits) {
        p.hist[blockIdx.x * p.digits + threadIdx.x] = count[threadIdx.x];
        if (p.next_hist) p.next_hist[blockIdx.x * p.digits + threadIdx.x] = 0;
    }
}

template <uint32_t ITEMS>
__global__ void __launch_bounds__(SORT_THREADS) embedding_move_kernel(const SortP p) {
    constexpr uint32_t TILE = SORT_THREADS * ITEMS;
    __shared__ uint32_t own[MAX_DIGITS], totals[MAX_DIGITS], before[MAX_DIGITS], scratch[SORT_WAVES];
    __shared__ uint16_t counts[SORT_WAVES * MAX_DIGITS];
    __shared__ uint32_t next[NEXT_COUNTS];
    if (blockIdx.x >= p.tiles) {
        clear_part(p, blockIdx.x - p.tiles);
        return;
    }
    if (p.next_hist)
        for (uint32_t i = threadIdx.x; i < p.tiles * p.digits; i += SORT_THREADS) next[i] = 0;
    const uint32_t tile = blockIdx.x;
    uint32_t key[ITEMS], pos[ITEMS], digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
        const uint32_t i = tile * TILE + item_index(ITEMS, k);
        key[k] = i < p.n ? (p.from_ids ? key_of(p, i) : p.key_in[i]) : 0;
        pos[k] = i < p.n ? (p.from_ids ? i : p.pos_in[i]) : 0;
        digit[k] = i < p.n ? (key[k] >> p.shift) & (p.digits - 1) : p.digits;
    }
    for (uint32_t i = threadIdx.x; i < SORT_WAVES * p.digits; i += SORT_THREADS) counts[i] = 0;
    if (threadIdx.x < p.digits) totals[threadIdx.x] = before[threadIdx.x] = 0;
    __syncthreads();
    // the tiles' counts of one digit are shared out over 1024 / digits threads
    {
        const uint32_t d = threadIdx.x & (p.digits - 1), part = threadIdx.x / p.digits, parts = SORT_THREADS / p.digits;
        uint32_t all = 0, front = 0;
        for (uint32_t t = part; t < p.tiles; t += parts) {
            const uint32_t x = p.hist[t * p.digits + d];
            all += x;
            if (t < tile) front += x;
        }
        atomicAdd(&totals[d], all);
        atomicAdd(&before[d], front);
    }
    rank_items<ITEMS>(digit, rank, counts, own, p.digits, ITEMS);
    prefix_digits(totals, scratch, p.digits);
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k)
        if (digit[k] < p.digits) {
            const uint32_t to = totals[digit[k]] + before[digit[k]] + rank[k];
            p.key_out[to] = key[k];
            p.pos_out[to] = pos[k];
            if (p.next_hist) atomicAdd(&next[to / TILE * p.digits + ((key[k] >> (p.shift + p.bits)) & (p.digits - 1))], 1u);
        }
    if (!p.next_hist) return;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.tiles * p.digits; i += SORT_THREADS)
        if (next[i]) atomicAdd(&p.next_hist[i], next[i]);
}

struct SumP {
    const float *gout;
    float *gtable, *part;  // part: [chunk][head, tail][E]
    const uint32_t *key, *pos;
    sg_rows g_rows;
    uint32_t n, E, V, chunk, chunks, pieces;
    float scale;
};

// Up to 128 tokens, in one launch: a workgroup owns some rows of the table, clears them, finds its tokens among all and sums
// the rows that have some in the tokens' order (23 tokens, table of 230 x 243: 5.4 us; 90 tokens, 2633 x 538: 10.8 us, with 30
// rows a workgroup instead of 4 15.6 us; 120 tokens, 30522 x 768: 20 us, 14 of them a fill's.  Sort, sums and join are three
// launches of 3.4 to 6.5 us at the least).
constexpr uint32_t FEW = 128, FEW_ROWS = 32, FEW_THREADS = 512;
struct FewP {
    const float *gout;
    const uint32_t *ids;
    float *gtable;
    sg_rows id_rows, g_rows;
    uint32_t n, E, V, rows;  // rows: what a workgroup owns, a multiple of 4
    uint32_t fill_vec;
    float scale;
};

template <bool NARROW>
__global__ void __launch_bounds__(FEW_THREADS) embedding_few_kernel(const FewP p) {
    __shared__ __attribute__((aligned(16))) uint32_t row_of[FEW];  // of each token, ~0: not here
    __shared__ uint32_t firsts[FEW], distinct;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t v0 = sg_workgroup() * p.rows;
    if (v0 >= p.V) return;
    const uint32_t rows = min(p.rows, p.V - v0);
    const uint32_t id = tid < p.n ? p.ids[sg_row_offset(p.id_rows, tid)] : ~0u;
    float *table = p.gtable + (uint64_t)v0 * p.E;
    const uint64_t total = (uint64_t)rows * p.E;
    for (uint64_t i = tid * 4u; i < total; i += FEW_THREADS * 4) {  // (whole tables of any E: a workgroup's rows begin at 16 bytes)
        if (p.fill_vec && i + 4 <= total) *reinterpret_cast<f32x4 *>(table + i) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        else for (uint64_t j = i; j < i + 4 && j < total; ++j) table[j] = 0.0f;
    }
    const bool here = id >= v0 && id - v0 < rows;
    const uint32_t row = here ? id - v0 : ~0u;
    if (tid < FEW) row_of[tid] = row;
    if (tid == 0) distinct = 0;
    if (!__syncthreads_or(here)) return;
    if (here) {
        bool first = true;
        for (uint32_t i = 0; i < tid; i += 4) {
            const uint4 o = *reinterpret_cast<const uint4 *>(&row_of[i]);
            first = first && o.x != row && (i + 1 >= tid || o.y != row) && (i + 2 >= tid || o.z != row) && (i + 3 >= tid || o.w != row);
        }
        if (first) firsts[atomicAdd(&distinct, 1u)] = row;  // in any order: the rows are summed each on its own
    }
    __syncthreads();  // the zeros, too, are written before the sums
    const uint32_t pieces = (p.E + 255) / 256, units = distinct * pieces;
    for (uint32_t u = wave; u < units; u += FEW_THREADS / 64) {  // a wavefront sums 256 columns of a row, 8 tokens in flight
        const uint32_t r = firsts[u / pieces], c = u % pieces * 256 + lane * 4;
        uint64_t a = __builtin_amdgcn_ballot_w64(row_of[lane] == r), b = __builtin_amdgcn_ballot_w64(row_of[64 + lane] == r);
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        while (a | b) {
            f32x4 x[8];
            uint32_t got = 0;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                if (!(a | b)) continue;
                const uint32_t token = a ? (uint32_t)__builtin_ctzll(a) : 64 + (uint32_t)__builtin_ctzll(b);
                if (a) a &= a - 1;
                else b &= b - 1;
                x[k] = load_cols<NARROW>(p.gout + sg_row_offset(p.g_rows, token), c, p.E);
                got = k + 1;
            }
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (k < got) acc += x[k];
        }
        store_cols<NARROW>(table + (uint64_t)r * p.E, c, p.E, acc * p.scale);
    }
}

// A wavefront sums 256 columns of one chunk of sorted tokens; BATCH rows are in flight at a time.  A large gout goes past
// the caches and leaves them to the table, which the next lookup reads (32768 tokens: that lookup 32 -> 20 us).
template <bool NARROW, bool NT, uint32_t BATCH>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const SumP p) {
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), lane = threadIdx.x & 63;
    if (unit >= p.chunks * p.pieces) return;
    const uint32_t chunk = unit / p.pieces, piece = unit - chunk * p.pieces;
    const uint32_t c = piece * 256 + lane * 4;
    const uint32_t first = chunk * p.chunk, last = min(first + p.chunk, p.n);
    const uint32_t own = min(first + lane, p.n - 1);
    const uint32_t key = p.key[own], pos = p.pos[own];
    const uint32_t prev = first > 0 ? p.key[first - 1] : ~0u, next = last < p.n ? p.key[last] : ~0u;  // no key is ~0
    bool from_before = prev == (uint32_t)__builtin_amdgcn_readfirstlane(key);
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t b = first; b < last; b += BATCH) {
        f32x4 x[BATCH];
        uint32_t id[BATCH + 1];
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k) {
            const uint32_t at = min(b + k, last - 1) - first;
            id[k] = (uint32_t)__builtin_amdgcn_readlane((int)key, (int)at);
            if (b + k < last && id[k] < p.V)
                x[k] = load_cols<NARROW, NT>(p.gout + sg_row_offset(p.g_rows, (uint32_t)__builtin_amdgcn_readlane((int)pos, (int)at)), c, p.E);
        }
        id[BATCH] = b + BATCH < last ? (uint32_t)__builtin_amdgcn_readlane((int)key, (int)(b + BATCH - first)) : next;
#pragma unroll
        for (uint32_t k = 0; k < BATCH; ++k) {
            if (b + k >= last || id[k] >= p.V) return;  // unknown tokens are the list's end
            acc += x[k];
            const bool end = b + k + 1 == last;
            const uint32_t follow = end ? next : id[k + 1];
            if (follow == id[k] && !end) continue;
            if (from_before) store_cols<NARROW>(p.part + (uint64_t)chunk * 2 * p.E, c, p.E, acc);
            else if (follow == id[k]) store_cols<NARROW>(p.part + ((uint64_t)chunk * 2 + 1) * p.E, c, p.E, acc);
            else store_cols<NARROW>(p.gtable + (uint64_t)id[k] * p.E, c, p.E, acc * p.scale);
            acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            from_before = false;
        }
    }
}

// A workgroup for 256 columns of the run that begins in a chunk and goes on behind it: the partial sums of the chunks it
// covers, shared out over the wavefronts in order and joined in order.
template <bool NARROW>
__global__ void __launch_bounds__(256) embedding_join_kernel(const SumP p) {
    __shared__ f32x4 sums[4][64];
    const uint32_t block = sg_workgroup(), chunk = block / p.pieces, piece = block - chunk * p.pieces;
    if (chunk + 1 >= p.chunks) return;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t c = piece * 256 + lane * 4;
    const uint32_t behind = (chunk + 1) * p.chunk;  // there is no work for the last chunk
    const uint32_t id = p.key[behind];
    if (id >= p.V || p.key[behind - 1] != id) return;                            // nothing goes on
    if (chunk > 0 && p.key[chunk * p.chunk - 1] == id) return;                   // it began further in front
    uint32_t lo = chunk + 1, hi = p.chunks - 1;  // the last chunk whose first token is of the run
    while (lo < hi) {
        const uint32_t mid = (lo + hi + 1) / 2;
        if (p.key[mid * p.chunk] == id) lo = mid;
        else hi = mid - 1;
    }
    const uint32_t count = lo - chunk, from = chunk + 1 + count * wave / 4, to = chunk + 1 + count * (wave + 1) / 4;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (wave == 0) acc = load_cols<NARROW>(p.part + ((uint64_t)chunk * 2 + 1) * p.E, c, p.E);
    uint32_t i = from;
    for (; i + 8 <= to; i += 8) {
        f32x4 x[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) x[k] = load_cols<NARROW>(p.part + (uint64_t)(i + k) * 2 * p.E, c, p.E);
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) acc += x[k];
    }
    for (; i < to; ++i) acc += load_cols<NARROW>(p.part + (uint64_t)i * 2 * p.E, c, p.E);
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) acc += sums[w][lane];
    store_cols<NARROW>(p.gtable + (uint64_t)id * p.E, c, p.E, acc * p.scale);
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
    p.scale = scale;
    const bool nt = sg_streaming((int64_t)p.n * E * 4);
    const uint64_t units = (uint64_t)p.n * p.pieces;
    sg_device_guard guard(ctx);
    const dim3 grid = sg_grid((units + 3) / 4);
    if (E < 4) hipLaunchKernelGGL((embedding_kernel<true, false>), grid, dim3(256), 0, ctx->stream, p);
    else if (nt) hipLaunchKernelGGL((embedding_kernel<false, true>), grid, dim3(256), 0, ctx->stream, p);
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
    SortP s{};
    s.ids = (const uint32_t *)ids->base + ids->offset;
    s.n = (uint32_t)sg_make_rows(ids, ids->rank, &s.id_rows);
    s.V = (uint32_t)gtable->extents[0];
    float *table = (float *)gtable->base + gtable->offset;
    const uint64_t table_floats = (uint64_t)s.V * E;
    SumP m{};
    m.gout = (const float *)gout->base + gout->offset;
    (void)sg_make_rows(gout, ids->rank, &m.g_rows);
    m.gtable = table;
    m.n = s.n;
    m.E = (uint32_t)E;
    m.V = s.V;
    m.scale = scale;
    m.pieces = (m.E + 255) / 256;
    if (s.n <= FEW) {
        FewP f{};
        f.gout = m.gout;
        f.ids = s.ids;
        f.gtable = table;
        f.id_rows = s.id_rows;
        f.g_rows = m.g_rows;
        f.n = s.n;
        f.E = m.E;
        f.V = s.V;
        f.scale = scale;
        // 512 workgroups or 64 KB of the table each, whichever is less, so that clearing fills the chip
        uint32_t rows = 16384 / f.E;
        rows = rows > FEW_ROWS ? FEW_ROWS : rows;
        rows = rows > (f.V + 511) / 512 ? (f.V + 511) / 512 : rows;
        f.rows = rows < 4 ? 4 : rows / 4 * 4;
        f.fill_vec = aligned16(table);
        sg_device_guard guard(ctx);
        const dim3 grid = sg_grid((s.V + f.rows - 1) / f.rows);
        if (E < 4) hipLaunchKernelGGL((embedding_few_kernel<true>), grid, dim3(FEW_THREADS), 0, ctx->stream, f);
        else hipLaunchKernelGGL((embedding_few_kernel<false>), grid, dim3(FEW_THREADS), 0, ctx->stream, f);
        SG_CHECK_LAUNCH(ctx, "embedding_grad");
        return SG_OK;
    }
    // Chunks short enough that their wavefronts fill the chip and none waits for rows twice (4096 tokens of 768: 8 a chunk 7.4 us,
    // 16 10.4 us; 32768 tokens: 16 a chunk 18.9 us and a join of 6.6, 32 28.8 and 6.4, 8 21.6 and 8.6), long enough that a run over
    // all tokens leaves few partial sums.  Sums and join together, 8 / 16 / 32 / 64 a chunk: 12000 tokens 19.3 / 21.7 / 31 / 48 us,
    // 20000 28.4 / 24.9 / 33.8 / 50, 50000 57 / 50.0 / 47.7 / 62, 100000 107 / 94 / 82.8 / 84.8, 200000 206 / 178 / 155 / 144,
    // 400000 405 / 344 / 306 / 275.
    m.chunk = s.n <= 16384 ? 8 : s.n <= 65536 ? 16 : s.n <= 262144 ? 32 : 64;
    m.chunks = (s.n + m.chunk - 1) / m.chunk;

    uint32_t bits = 1;
    while ((s.V >> bits) != 0) ++bits;  // keys are 0..V
    s.passes = (bits + 8) / 9;
    s.bits = (bits + s.passes - 1) / s.passes;
    s.digits = 1u << s.bits;
    const bool single = s.n <= SINGLE;
    const uint32_t items = s.n <= 131072 ? 2 : 4, tile = SORT_THREADS * items;
    s.tiles = single ? 1 : (s.n + tile - 1) / tile;
    // the sorted list, a second one to move between where there are several launches, the tiles' counts, the partial sums
    const uint64_t list = (uint64_t)(s.n + 3) / 4 * 4, counts = single ? 0 : 2 * (uint64_t)s.tiles * s.digits;
    const uint64_t words = list * (single ? 2 : 4) + (counts + 3) / 4 * 4 + (uint64_t)m.chunks * 2 * E;
    sg_device_guard guard(ctx);
    sg_workspace space(ctx);
    if ((rc = space.take(words * 4)) != SG_OK) return rc;
    uint32_t *key[2], *pos[2], *w = (uint32_t *)space.p;
    key[0] = w;
    pos[0] = w + list;
    key[1] = single ? nullptr : w + 2 * list;
    pos[1] = single ? nullptr : w + 3 * list;
    w += list * (single ? 2 : 4);
    s.hist = w;
    m.part = (float *)(w + (counts + 3) / 4 * 4);

    const uint64_t per_block = (uint64_t)SORT_THREADS * FILL * 4, fill_blocks = (table_floats + per_block - 1) / per_block;
    s.fill_vec = aligned16(table);
    if (single) {
        s.key_out = key[0];
        s.pos_out = pos[0];
        s.fill = table;
        s.fill_floats = table_floats;
        const dim3 grid((unsigned)(1 + fill_blocks));
        if (s.n <= SORT_THREADS) hipLaunchKernelGGL((embedding_sort_kernel<1>), grid, dim3(SORT_THREADS), 0, ctx->stream, s);
        else if (s.n <= SORT_THREADS * 4) hipLaunchKernelGGL((embedding_sort_kernel<4>), grid, dim3(SORT_THREADS), 0, ctx->stream, s);
        else hipLaunchKernelGGL((embedding_sort_kernel<8>), grid, dim3(SORT_THREADS), 0, ctx->stream, s);
        SG_CHECK_LAUNCH(ctx, "embedding_grad sort");
        m.key = key[0];
        m.pos = pos[0];
    } else {
        // every launch clears its share of the table
        const bool fused = (uint64_t)s.tiles * s.digits <= NEXT_COUNTS && s.passes == 2;
        const uint32_t launches = fused ? 3 : 2 * s.passes;
        const uint64_t share = (fill_blocks + launches - 1) / launches;
        uint64_t cleared = 0;
        uint32_t *const hist[2] = {s.hist, s.hist + (uint64_t)s.tiles * s.digits};
        auto take_share = [&]() {
            const uint64_t at = cleared * per_block;
            const uint64_t blocks = cleared + share <= fill_blocks ? share : fill_blocks - cleared;
            s.fill = table + at;
            s.fill_floats = blocks * per_block <= table_floats - at ? blocks * per_block : table_floats - at;
            cleared += blocks;
            return dim3((unsigned)(s.tiles + blocks));
        };
        for (uint32_t pass = 0; pass < s.passes; ++pass) {
            s.from_ids = pass == 0;
            s.shift = pass * s.bits;
            s.key_in = key[(pass + 1) & 1];
            s.pos_in = pos[(pass + 1) & 1];
            s.key_out = key[pass & 1];
            s.pos_out = pos[pass & 1];
            s.hist = hist[fused ? pass : 0];
            s.next_hist = fused && pass == 0 ? hist[1] : nullptr;
            if (!fused || pass == 0) {
                const dim3 count_grid = take_share();
                if (items == 2) hipLaunchKernelGGL((embedding_count_kernel<2>), count_grid, dim3(SORT_THREADS), 0, ctx->stream, s);
                else hipLaunchKernelGGL((embedding_count_kernel<4>), count_grid, dim3(SORT_THREADS), 0, ctx->stream, s);
                SG_CHECK_LAUNCH(ctx, "embedding_grad count");
            }
            const dim3 move_grid = take_share();
            if (items == 2) hipLaunchKernelGGL((embedding_move_kernel<2>), move_grid, dim3(SORT_THREADS), 0, ctx->stream, s);
            else hipLaunchKernelGGL((embedding_move_kernel<4>), move_grid, dim3(SORT_THREADS), 0, ctx->stream, s);
            SG_CHECK_LAUNCH(ctx, "embedding_grad move");
        }
        m.key = s.key_out;
        m.pos = s.pos_out;
    }
    const bool narrow = E < 4, nt = sg_streaming((int64_t)m.n * E * 4);
    const dim3 sum_grid((m.chunks * m.pieces + 3) / 4), join_grid = sg_grid((uint64_t)(m.chunks - 1) * m.pieces);
    if (narrow) hipLaunchKernelGGL((embedding_sum_kernel<true, false, 4>), sum_grid, dim3(256), 0, ctx->stream, m);
    else if (nt) hipLaunchKernelGGL((embedding_sum_kernel<false, true, 16>), sum_grid, dim3(256), 0, ctx->stream, m);
    else hipLaunchKernelGGL((embedding_sum_kernel<false, false, 16>), sum_grid, dim3(256), 0, ctx->stream, m);
    SG_CHECK_LAUNCH(ctx, "embedding_grad sums");
    if (m.chunks > 1) {
        if (narrow) hipLaunchKernelGGL((embedding_join_kernel<true>), join_grid, dim3(256), 0, ctx->stream, m);
        else hipLaunchKernelGGL((embedding_join_kernel<false>), join_grid, dim3(256), 0, ctx->stream, m);
        SG_CHECK_LAUNCH(ctx, "embedding_grad join");
    }
    return SG_OK;
}
