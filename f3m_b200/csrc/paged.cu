// A cache of keys and values in pages: new tokens appended, their attention over it, accepted paths of drafted trees.
#include <algorithm>
#include "seq.cuh"

namespace f3m {

// ---- new tokens to their pages ----------------------------------------------------------------------------------------------
// A CTA has AP_TOKENS neighbouring tokens of a sequence.  Their places and angles are taken once for all heads: the part of a whole turn is position * turns modulo
// 2^64, exact for any position, and what is left, in FP32, is at most half a turn.  Then its rows, (token, head) of queries, keys and values, 16 lanes or 8 to a row with 16 bytes
// each; a lane's partner in a half-split rotation hands its columns over.  Memory is the bound: every array is read and written once.  10121 tokens in 8 chunks, 32 heads and 8, width
// 128: 52-56 us, 4.8 TB/s, 73 % of the measured copy (four tokens a CTA 64; a thread's vectors found by divisions 62; four of them in flight 92).
constexpr int AP_TOKENS = 2, AP_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(AP_THREADS, 8) append_tokens(const __grid_constant__ AppendArgs a) {
    __shared__ int slot_s[AP_TOKENS], pos_s[AP_TOKENS], page_s[AP_TOKENS];
    __shared__ __align__(16) float2 turn_s[AP_TOKENS][F3M_MAX_WIDTH / 2];   // cosines and sines, two pairs of each lane side by side, then the lanes' next two
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, blockIdx.x)];
    const int i0 = e.z + AP_TOKENS * blockIdx.y, m = min(AP_TOKENS, min(e.z + SEQ_TILE, e.y) - i0), half = a.rotation.columns / 2;
    const int own = a.rotation.interleaved ? 4 : 8, turned = half / own;   // pairs of a lane, lanes with pairs of their own
    if (m <= 0) return;
    if (threadIdx.x < m) {
        const int i = i0 + threadIdx.x, length = paged_length(a.c, e.w);
        int depth = i;
        if (a.parents) {
            const int *parents = a.parents + e.x;
            depth = 0;
            for (int p = parent_of(parents, i); p >= 0; p = parent_of(parents, p)) depth++;
        }
        slot_s[threadIdx.x] = length + i;
        pos_s[threadIdx.x] = length + depth;
        page_s[threadIdx.x] = paged_page(a.c, e.w, (int64_t)length + i);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < m * half; x += AP_THREADS) {
        const int t = x / half, i = x % half;
        const int64_t part = (int64_t)((uint64_t)pos_s[t] * a.rotation.turns[i]);   // of a whole turn, 2^64; as signed the nearest one
        float s, c;
        sincospif(0x1p-63f * (float)part, &s, &c);
        turn_s[t][i % own / 2 * 2 * turned + 2 * (i / own) + (i & 1)] = make_float2(c, s);
    }
    __syncthreads();
    const int lanes = a.c.width > 64 ? 16 : 8, step = AP_THREADS / lanes, c = threadIdx.x & (lanes - 1), per_token = a.heads + 2 * a.c.kv_heads;
    const bool inside = 8 * c < a.c.width, split = !a.rotation.interleaved, second = 8 * c >= half;
    const bool turns = 8 * c < 2 * half;
    const int partner = (threadIdx.x & 31) + (second ? -half : half) / 8, at = 2 * (split && second ? c - turned : c);
    int t = 0, j = threadIdx.x / lanes;
    for (int r = 0; r < m * per_token; r += step, j += step) {   // whole warps
        while (j >= per_token) { j -= per_token; t++; }
        const bool query = j < a.heads, value = j >= a.heads + a.c.kv_heads;
        const int h = query ? j : value ? j - a.heads - a.c.kv_heads : j - a.heads;
        uint16_t *dst = nullptr;
        uint4 f = make_uint4(0u, 0u, 0u, 0u);
        if (t < m && inside) {
            const int64_t row = e.x + i0 + t;
            if (query) dst = reinterpret_cast<uint16_t *>(a.q_out.data) + row * a.q_out.token_stride + (int64_t)h * a.q_out.head_stride + 8 * c;
            else if (page_s[t] >= 0) {
                const f3m_pages &p = value ? a.c.v : a.c.k;
                dst = reinterpret_cast<uint16_t *>(p.data) + paged_at(a.c, p, page_s[t], slot_s[t], h) + 8 * c;
            }
            const f3m_rows &from = query ? a.q : value ? a.v : a.k;
            f = *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(from.data) + row * from.token_stride + (int64_t)h * from.head_stride + 8 * c);
        }
        uint32_t x[4] = {f.x, f.y, f.z, f.w}, y[4];
        if (split && half)
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = __shfl_sync(0xffffffffu, x[i], partner & 31);
        if (turns && !value && t < m) {
            const float4 *turn = reinterpret_cast<const float4 *>(turn_s[t] + at);   // cosine and sine, of two pairs
            if (split) {   // x cos - y sin, and of the second half x cos + y sin
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 v = Half<T>::unpack(x[i]), w = Half<T>::unpack(y[i]);
                    const float4 p = turn[i * turned];
                    const float s0 = second ? p.y : -p.y, s1 = second ? p.w : -p.w;
                    x[i] = Half<T>::pack(v.x * p.x + w.x * s0, v.y * p.z + w.y * s1);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float2 v = Half<T>::unpack(x[i]), w = Half<T>::unpack(x[i + 1]);
                    const float4 p = turn[i / 2 * turned];
                    x[i] = Half<T>::pack(v.x * p.x - v.y * p.y, v.x * p.y + v.y * p.x);
                    x[i + 1] = Half<T>::pack(w.x * p.z - w.y * p.w, w.x * p.w + w.y * p.z);
                }
            }
        }
        if (dst) *reinterpret_cast<uint4 *>(dst) = make_uint4(x[0], x[1], x[2], x[3]);
    }
}

void paged_append(int type, const AppendArgs &a, cudaStream_t s) {
    const dim3 grid(a.s.tiles, (std::min(a.s.longest, SEQ_TILE) + AP_TOKENS - 1) / AP_TOKENS);
    if (type == F3M_TYPE_BF16) append_tokens<__nv_bfloat16><<<grid, AP_THREADS, 0, s>>>(a);
    else append_tokens<__half><<<grid, AP_THREADS, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}

// ---- attention of new tokens ------------------------------------------------------------------------------------------------
// An item is one key head and new tokens of a sequence whose rows, (token, head) of the heads that share it, fill one tile of 128 or two; it walks over the tiles of 128
// keys that some of its rows see.  Items of one tile of rows (one token, a drafted tree) are memory's: two CTAs an SM, so that one's weights are taken while the
// other's copies and products run, also where items are short.  Items of two (chunks of prompts) are arithmetic's: a CTA an SM, two tiles of rows that share each
// tile of keys.  How long a sequence is stands on the device only, so that each CTA counts for itself: CTA c of G takes the share c U / G .. (c + 1) U / G of all items' U
// tiles, cuts through items where that falls, and paged_join puts the parts together, in one order.
//
// What bounds it: of one token for 32 sequences up to 16384, 32 heads on 8, width 128, memory (176-206 us, 5.1-5.9 TB/s of 6.5); of trees of 32 tokens on the same, 215-238 us, shared memory and
// the chain of a tile (scores, read twice, maximum, exponentials, product): beside more than 40 rows of width 128 half an SM's holds two slots, one of keys and one of values, so that a copy waits for the
// product with what was there before (trees of 8 tokens 181 us, 10: 185, 11: 200), and more warps with rows take longer (16: 208, 20: 222, 32: 231).  Of chunks of 2048
// and 1021 tokens, window 4096, it is that chain: 320-331 us, 0.62-0.65 PFLOP/s (0.82-0.85 where all is seen).
//
// Heads that do not divide 128 evenly pay for the entries of 256 tokens that an item does not cross: 3 to a key head make items of 84, 84, 84 and 4 tokens, the last in the other kernel (chunks that see
// all: 0.67 PFLOP/s with 3, 0.76 with 5, 0.83-0.85 with 4 and 8).  Widths are taken in blocks of 64 columns: 80 costs what 128 does (470 us, 489), and rows that do not start on whole lines
// more than that (one token: 206 us with 80, 176 with 128).
//
// As in window attention S = Q K^T goes to tensor memory, a thread takes the weights of one row and writes them over S, from where they go into O += P V: rounded to 16 bits, as the product
// takes them, which is as much as an output's own rounding; the row's sum is of those before.
//
// Keys that only a part of the item's rows sees (the window's edge, new tokens, a tree, missing pages) go by bits, a word for 32 of them.  A value that is not finite would
// reach every row there, as zero times it: it is taken out of the tile, and added to the rows that see it when they have been written (poison_row).
constexpr int PG_BLOCK = SEQ_TILE * 128, PG_RING = 4, PG_THERE = 8, PG_MAX_SLOTS = 8;
// What an item takes beside its tiles of keys, in tiles: of one tile of rows 2 (trees of 32 tokens for 32 sequences 237 us, 250 with 1, 236 with 4; 96 single tokens on up to 3800
// 144, 142, 146), of two tiles 1 (chunks 331 us, 330 with 2, 328 with 4).
template <int TILES> constexpr int PG_ITEM = TILES == 1 ? 2 : 1;
constexpr float PG_NO_SUM = 0x1p60f;   // some exponent was not a number (exp2_poly)
constexpr float PG_MET = 0x1p-126f;    // a row's sum is at least this if it has seen a key; of a tile that all see the polynomial's least, 2^-125, comes to more
constexpr float PG_ALL_LOW = -1.f;     // in the place of a part's sum: it has seen keys, and all their scores are -inf
constexpr int PG_WORDS = F3M_TREE_MAX / 32;

struct PagedItem {
    int row0, n, b, i0, tokens, length;   // the sequence's first row, new tokens, number; first token of the item, how many; tokens in the cache
    int kv_head, sinks, first, keys;      // tiles of keys: the first `sinks` of the sequence, then those from tile `first` on; `keys` in all
    __device__ __forceinline__ int key(int j) const { return SEQ_TILE * (j < sinks ? j : first + j - sinks); }
    template <int TILES> __device__ __forceinline__ int cost() const { return keys ? keys + PG_ITEM<TILES> : 0; }   // the item's own comes behind its last tile
};
struct PagedPart {   // of an item: tiles of keys j0 .. j1 - 1
    PagedItem w;
    int j0, j1, slot;   // slot: where its sums go; -1: all of the item, the outputs themselves
};
struct PagedSplit {   // an item whose first part is the last one of a CTA
    PagedItem w;
    int parts;   // 0: none
};
struct PagedKernel {
    PagedArgs a;
    CUtensorMap mq, mk, mv;
    int group, tokens;     // heads that share a key head; tokens of a tile of rows
    int subs, entries;     // items of 256 tokens of a sequence, of all sequences
    int page_shift, box;   // box: tokens of a copy
    int q_box, q_rows, places, slots;   // rows of a copy, rows that are kept of a tile's 128 (the products take whatever lies behind them for the others), places for these, for keys or values
    int rows;              // of a part's place in the workspace
    bool wide;
    float c;               // |scale| log2(e)
    float2 *stat;          // (2 G, rows): maximum, sum of weights
    float *sums;           // (2 G, rows, width)
    PagedSplit *split;     // (G)
    int *err;
};

// Entry e: a sequence's tokens, without a key head; no tiles: none are left, or another kernel has them
template <int TILES>
__device__ __forceinline__ PagedItem paged_item(const PagedKernel &p, int e) {
    const PagedArgs &a = p.a;
    const int4 q = reinterpret_cast<const int4 *>(a.s.table)[seq_pair_by_past(a.s, e / p.subs)];
    PagedItem w;
    w.row0 = q.x; w.n = q.y; w.b = q.w;
    const int in = 2 * p.tokens * (e % p.subs);
    w.i0 = q.z + in;
    w.tokens = max(0, min(min(2 * p.tokens, 2 * SEQ_TILE - in), w.n - w.i0));
    w.length = paged_length(a.c, w.b);
    w.kv_head = 0;
    // the first new token that a row may be, by its position: a tree's may be a root
    w.first = max(0, w.length + (a.parents ? 0 : w.i0) - a.window + 1) / SEQ_TILE;
    w.sinks = min((a.sinks + SEQ_TILE - 1) / SEQ_TILE, w.first);
    w.keys = w.tokens && (w.tokens > p.tokens) == (TILES == 2) ? w.sinks + (w.length + w.i0 + w.tokens - 1) / SEQ_TILE - w.first + 1 : 0;
    return w;
}
// Whether all rows of the item see all keys of a tile, if they have pages
__device__ __forceinline__ bool seen_by_all(const PagedArgs &a, const PagedItem &w, int key) {
    const int last = w.length + w.i0 + w.tokens - 1;   // the furthest position
    return key + SEQ_TILE - 1 <= w.length + (a.parents ? -1 : w.i0) && (last - key < a.window || key + SEQ_TILE <= a.sinks);
}
__device__ __forceinline__ uint32_t ones(int from, int to) {   // bits from .. to - 1 of a word
    from = max(from, 0);
    to = min(to, 32);
    return to > from ? (0xffffffffu >> (32 - to + from)) << from : 0u;
}
// The keys from `at` to at + 31 that a row at position pos sees; `there`: which of their four groups of 8 have a page.  up: its last key but for a tree's; above: a tree's
// new tokens that it sees, from place `length` on
__device__ __forceinline__ uint32_t seen_keys(const PagedArgs &a, int length, int at, uint32_t there, int pos, int up, const uint32_t *above) {
    uint32_t m = (ones(pos - a.window + 1 - at, 32) | ones(0, a.sinks - at)) & ones(0, up + 1 - at);
    if (above) {
        const int bit = at - length, k = bit >> 5;
        const uint32_t lo = k >= 0 && k < PG_WORDS ? above[k] : 0u, hi = k >= -1 && k + 1 < PG_WORDS ? above[k + 1] : 0u;
        m |= __funnelshift_r(lo, hi, bit & 31);
    }
    const uint32_t groups = (there & 1u) | (there & 2u) << 7 | (there & 4u) << 14 | (there & 8u) << 21;
    return m & groups * 0xffu;
}
__device__ __forceinline__ bool finite16(uint32_t v, uint32_t exponent) { return (v & exponent) != exponent; }   // the lower half of a word

// Tiles of a part are noted in a word: a bit for each, or for 2^shift next to one another where there are more than 32
__device__ __forceinline__ int tile_shift(const PagedPart &part) { return max(27 - __clz(part.j1 - part.j0 - 1), 0); }

// Values that are not finite, of keys in tiles that were cleared of them, to the columns of a row that sees them.  Only tiles noted in `bad` are looked at: in a cache with pages missing
// everywhere all tiles are cleared ones, and one such value would have a row read all of them again (32 sequences of 16384, a page in 8 missing: 1.1 ms, all tiles read 105, without the value 0.54).
template <typename T, typename O>
__device__ __noinline__ void poison_row(const PagedKernel &p, const PagedPart &part, uint32_t bad, int pos, int up, const uint32_t *above, O *row) {
    const PagedArgs &a = p.a;
    const PagedItem &w = part.w;
    constexpr uint32_t exponent = Half<T>::type == F3M_TYPE_BF16 ? 0x7f80u : 0x7c00u;
    const int shift = tile_shift(part);
    for (int j = part.j0; j < part.j1; j++) {
        if (!(bad >> ((j - part.j0) >> shift) & 1u)) continue;
        const int key = w.key(j);
        uint32_t there = 0;
        for (int g = 0; g < SEQ_TILE / 8; g++) there |= (uint32_t)(paged_page(a.c, w.b, (int64_t)key + 8 * g) >= 0) << g;
        if (there == 0xffffu && seen_by_all(a, w, key)) continue;
        for (int q = 0; q < 4; q++)
            for (uint32_t m = seen_keys(a, w.length, key + 32 * q, there >> 4 * q, pos, up, above); m; m &= m - 1) {
                const int64_t slot = key + 32 * q + __ffs(m) - 1;
                const uint16_t *v = reinterpret_cast<const uint16_t *>(a.c.v.data) + paged_at(a.c, a.c.v, paged_page(a.c, w.b, slot), slot, w.kv_head);
                for (int c = 0; c < a.c.width; c += 32) {   // four loads on their way
                    uint4 f[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) f[i] = c + 8 * i < a.c.width ? *reinterpret_cast<const uint4 *>(v + c + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
                    bool finite = true;
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        for (uint32_t x : {f[i].x, f[i].y, f[i].z, f[i].w}) finite &= finite16(x, exponent) && finite16(x >> 16, exponent);
                    if (finite) continue;
#pragma unroll 1
                    for (int i = c; i < min(c + 32, a.c.width); i++) {
                        const float y = Half<T>::unpack(v[i]).x;
                        if (isfinite(y)) continue;
                        if constexpr (sizeof(O) == 4) row[i] += y;
                        else row[i] = (O)Half<T>::pack(Half<T>::unpack(row[i]).x + y, 0.f);
                    }
                }
            }
    }
}

template <typename T, int NB, int TILES>
__global__ void __launch_bounds__(128 * TILES + 64, 3 - TILES) paged_tiles(const __grid_constant__ PagedKernel p) {
    constexpr int ROWS = 128 * TILES, THREADS = ROWS + 64, WARPS = THREADS / 32, COPY = 4 * TILES, PRODUCTS = COPY + 1;
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * PG_MAX_SLOTS + 2 * PG_RING + 16];
    __shared__ PagedPart ring_s[PG_RING];
    __shared__ long long warp_s[WARPS], start_s[2];
    __shared__ uint32_t tmem_s, bad_s[2][4], there_s[PG_THERE];
    __shared__ int gave_up_s, go_s[2];
    __shared__ int16_t parent_s[F3M_TREE_MAX], depth_s[ROWS];
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, slots = p.slots;
    // the new tokens that each token sees; rows, in one or two places, or two tiles side by side; tiles of keys and values
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u;
    uint32_t(*above_s)[PG_WORDS] = reinterpret_cast<uint32_t(*)[PG_WORDS]>(raw + (smem - tc::smem_u32(raw)));
    const uint32_t q_at = smem + ROWS * PG_WORDS * 4, q_block = p.q_rows * 128, slots_at = q_at + p.places * NB * q_block;
    auto q_tile = [&](int place) { return q_at + place * NB * q_block; };
    auto slot_tile = [&](int s) { return slots_at + s * NB * PG_BLOCK; };
    auto place_of = [&](int part, int t) { return TILES == 2 ? t : part & (p.places - 1); };   // of a part's rows, and how often it was used before
    auto use_of = [&](int part) { return TILES == 1 && p.places == 2 ? part >> 1 : part; };

    if (warp == COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 256 * TILES);
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = b_full + 8 * PG_MAX_SLOTS, b_part = b_free + 8 * PG_MAX_SLOTS, b_part_free = b_part + 8 * PG_RING, b_q = b_part_free + 8 * PG_RING,
                   b_q_free = b_q + 16, b_s = b_q + 32, b_p = b_q + 48, b_p2 = b_q + 64, b_o = b_q + 80, b_o_read = b_q + 96, b_none = b_q + 104, b_clear = b_q + 112;
    if (tid == 0) {
        for (int i = 0; i < 2 * PG_MAX_SLOTS; i++) tc::mbar_init(b_full + 8 * i, 1);   // landed, free
        for (int i = 0; i < PG_RING; i++) {
            tc::mbar_init(b_part + 8 * i, 1);                                          // a part is told
            tc::mbar_init(b_part_free + 8 * i, WARPS - 1);                             // and done with, by all warps but one
        }
        for (int t = 0; t < 2; t++) {
            tc::mbar_init(b_q + 8 * t, 1);       // a tile of rows landed, free
            tc::mbar_init(b_q_free + 8 * t, 1);
            tc::mbar_init(b_s + 8 * t, 1);       // S ready
            tc::mbar_init(b_p + 8 * t, 128);     // weights of the first 64 keys written
            tc::mbar_init(b_p2 + 8 * t, 128);    // of the other 64
            tc::mbar_init(b_o + 8 * t, 1);       // O ready
            tc::mbar_init(b_clear + 8 * t, 4);   // values of a tile that is seen in part are finite, of one such tile and of the next
        }
        tc::mbar_init(b_o_read, ROWS);
        tc::mbar_init(b_none, 1);                // no products in flight
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    // tiles of all items, and where this CTA's begin
    auto cost_of = [&](int e) { return e < p.entries ? (long long)paged_item<TILES>(p, e).template cost<TILES>() * a.c.kv_heads : 0ll; };
    auto scan = [&](long long v, long long &all) {   // of the block's threads: the sum up to this one, and of all
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += y;
        }
        __syncthreads();
        if (lane == 31) warp_s[warp] = v;
        __syncthreads();
        all = 0;
        long long before = 0;
        for (int i = 0; i < WARPS; i++) {
            if (i == warp) before = all;
            all += warp_s[i];
        }
        return v + before;
    };
    long long total = 0, mine = 0, up_to = 0, sum_of = 0;
    for (int e = 0; e < p.entries; e += THREADS) {
        mine = cost_of(e + tid);
        up_to = scan(mine, sum_of);
        total += sum_of;
    }
    const int ctas = (int)min((long long)gridDim.x, total), cta = blockIdx.x;   // a tile at least for each
    const long long u0 = cta < ctas ? cta * total / ctas : total, u1 = cta < ctas ? (cta + 1) * total / ctas : total;
    long long base = 0;
    for (int e = 0; e < p.entries; e += THREADS) {
        if (p.entries > THREADS) {
            mine = cost_of(e + tid);
            up_to = scan(mine, sum_of);
        }
        if (u0 < base + up_to && u0 >= base + up_to - mine) { start_s[0] = e + tid; start_s[1] = u0 - (base + up_to - mine); }
        base += sum_of;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s, t_out = tmem + ROWS;

    if (warp == COPY) {
        // ---- parts told to the others, copies, K V K V ..: without a stop between parts; a lane has a page of a tile ----
        int x = 0, parts = 0, e = u0 < u1 ? (int)start_s[0] : 0, e0 = e, rows_told = 0;   // copies, parts, parts whose rows are on their way so far
        long long left = u1 - u0;
        bool stop = false;   // of the whole warp
        const int boxes = SEQ_TILE / p.box;
        const uint32_t page_mask = (1u << p.page_shift) - 1;
        auto wait_all = [&](uint32_t bar, uint32_t parity) {
            wait(bar, parity);
            stop = __any_sync(0xffffffffu, gave_up_s);
        };
        // entries are read 32 at a time, a lane each
        PagedItem held = paged_item<TILES>(p, min(e + lane, p.entries - 1)), w;
        auto entry = [&](int i) {
            if (i - e0 >= 32) {
                e0 = i;
                held = paged_item<TILES>(p, min(i + lane, p.entries - 1));
            }
            auto same = [&](int v) { return __shfl_sync(0xffffffffu, v, i - e0); };
            return PagedItem{same(held.row0), same(held.n), same(held.b), same(held.i0), same(held.tokens), same(held.length), 0, same(held.sinks), same(held.first), same(held.keys)};
        };
        auto page_at = [&](const PagedItem &z, int k) { return lane < boxes ? paged_page(a.c, z.b, (int64_t)z.key(k) + lane * p.box) : -1; };
        w = entry(e);
        int j = 0;
        if (left) { w.kv_head = min((int)(start_s[1] / w.template cost<TILES>()), a.c.kv_heads - 1); j = (int)(start_s[1] % w.template cost<TILES>()); }
        if (lane == 0) p.split[cta].parts = 0;
        auto next = [&] {   // the item behind this one
            left -= min(left, (long long)w.template cost<TILES>() - j);
            j = 0;
            if (left && ++w.kv_head == a.c.kv_heads)
                do {
                    if (++e == p.entries) left = 0;
                    else w = entry(e);
                } while (left && w.keys == 0);
        };
        if (left && j >= w.keys) next();
        int page = left ? page_at(w, j) : -1;
        while (left > 0) {
            const int r = parts % PG_RING, j0 = j, j1 = (int)min((long long)w.keys, j + left);
            if (parts >= PG_RING) wait_all(b_part_free + 8 * r, (parts / PG_RING - 1) & 1);
            if (stop) break;
            if (lane == 0) {
                ring_s[r] = PagedPart{w, j0, j1, j0 > 0 || j1 < w.keys ? 2 * cta + (j0 == 0) : -1};
                if (j0 == 0 && j1 < w.keys)   // the item's last tile is keys - j1 behind this CTA's
                    p.split[cta] = {w, (int)(((u1 + w.keys - j1) * ctas - 1) / total) - cta + 1};
                tc::mbar_arrive(b_part + 8 * r);
            }
            __syncwarp();
            const PagedItem &now = ring_s[r].w;
            next();
            const int later = left ? page_at(w, 0) : -1;   // of the next part
            for (int t = 0; t < TILES; t++) {
                const int place = place_of(parts, t), use = use_of(parts);
                if (use) wait_all(b_q_free + 8 * place, (use - 1) & 1);
                if (stop) break;
                if (lane == 0) {
                    tc::mbar_expect_tx(b_q + 8 * place, NB * p.q_box * 128);
                    for (int c = 0; c < NB; c++)
                        tc::tma_rows(q_tile(place) + c * q_block, &p.mq, 64 * c, now.kv_head * p.group, now.row0 + now.i0 + t * p.tokens, b_q + 8 * place);
                }
                rows_told = parts + 1;
            }
            for (int k = j0; k < j1 && !stop; k++) {
                const int at = page, row = (int)((uint32_t)(now.key(k) + lane * p.box) & page_mask);
                uint32_t there = __ballot_sync(0xffffffffu, at >= 0);
                there = __ballot_sync(0xffffffffu, lane < SEQ_TILE / 8 && there >> (8 * lane / p.box) & 1u);   // of 16 groups of 8 keys
                page = k + 1 < j1 ? page_at(now, k + 1) : later;
                for (int v = 0; v < 2; v++, x++) {
                    const int s = x % slots;
                    if (x >= slots) wait_all(b_free + 8 * s, (x / slots - 1) & 1);
                    if (stop) break;
                    if (lane == 0) {
                        if (v == 0) there_s[x / 2 % PG_THERE] = there;
                        tc::mbar_expect_tx(b_full + 8 * s, NB * PG_BLOCK);
                    }
                    __syncwarp();
                    if (lane < boxes)   // of a page that is not there zeros come
                        for (int c = 0; c < NB; c++)
                            tc::tma_page(slot_tile(s) + c * PG_BLOCK + lane * p.box * 128, v ? &p.mv : &p.mk, 64 * c, now.kv_head, row, at, b_full + 8 * s);
                }
            }
            parts++;
            if (stop) break;
        }
        const int r = parts % PG_RING;
        if (!stop && parts >= PG_RING) wait_all(b_part_free + 8 * r, (parts / PG_RING - 1) & 1);
        if (lane == 0) {
            if (!stop) {   // no more parts
                ring_s[r].j1 = 0;
                tc::mbar_arrive(b_part + 8 * r);
            }
            for (int s = 0; s < slots; s++)   // the last copies
                if (x > s) wait.drain(b_full + 8 * s, ((x - 1 - s) / slots) & 1);
            for (int part = max(0, rows_told - (TILES == 2 ? 1 : p.places)); part < rows_told; part++)   // each place's last
                for (int t = 0; t < TILES; t++) wait.drain(b_q + 8 * place_of(part, t), use_of(part) & 1);
        }
    } else if (warp == PRODUCTS) {
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        // a negative scale turns S's sign: bit 13 negates A
        const uint32_t i_s = tc::idesc_f16(bf, 128, 128, false, false) | (a.scale < 0.f ? 1u << 13 : 0u), i_o = tc::idesc_f16(bf, 128, 64 * NB, false, true);
        int x = 0, np = 0;
        for (int parts = 0;; parts++) {
            const int r = parts % PG_RING;
            wait(b_part + 8 * r, (parts / PG_RING) & 1);
            if (__any_sync(0xffffffffu, gave_up_s)) break;
            const int keys = ring_s[r].j1 - ring_s[r].j0, end = ring_s[r].j1;
            __syncwarp();
            if (end == 0) break;
            if (lane == 0) tc::mbar_arrive(b_part_free + 8 * r);
            auto scores = [&](int t, int k) {
                const int at = x + 2 * k, s = at % slots, place = place_of(parts, t);
                wait(b_full + 8 * s, (at / slots) & 1);
                tc::fence_after_sync();
                if (tc::elect()) {
#pragma unroll
                    for (int i = 0; i < NB; i++) tc::product64<2, 2>(tmem + 128 * t, tc::desc_k(q_tile(place) + i * q_block), tc::desc_k(slot_tile(s) + i * PG_BLOCK), i_s, i);
                    tc::mma_commit(b_s + 8 * t);
                    if (t == TILES - 1) tc::mma_commit(b_free + 8 * s);
                    if (k == keys - 1) tc::mma_commit(b_q_free + 8 * place);
                }
            };
            for (int t = 0; t < TILES; t++) {
                wait(b_q + 8 * place_of(parts, t), use_of(parts) & 1);
                scores(t, 0);
            }
            if (parts) wait(b_o_read, (parts - 1) & 1);
            for (int k = 0; k < keys; k++) {
                const int at = x + 2 * k + 1, sv = at % slots;
                const bool more = k + 1 < keys;
                wait(b_full + 8 * sv, (at / slots) & 1);
                for (int t = 0; t < TILES; t++) {
                    wait(b_p + 8 * t, np & 1);
                    tc::fence_after_sync();
                    if (tc::elect()) tc::product_tmem64(t_out + 128 * t, tmem + 128 * t, slot_tile(sv), i_o, k > 0);
                    wait(b_p2 + 8 * t, np & 1);
                    tc::fence_after_sync();
                    if (tc::elect()) {
                        tc::product_tmem64(t_out + 128 * t, tmem + 128 * t + 32, slot_tile(sv) + 64 * 128, i_o, 1);
                        if (t == TILES - 1) tc::mma_commit(b_free + 8 * sv);
                        if (!more) tc::mma_commit(b_o + 8 * t);
                    }
                    if (more) scores(t, k + 1);
                }
                np++;
            }
            x += 2 * keys;
        }
        wait.drain_products(b_none);
    } else {
        // ---- weights: thread r of a tile has its row r ----
        const int t = warp >> 2, r = tid & 127, wq = warp & 3, in = r / p.group, head = r % p.group;
        const uint32_t lanes = (uint32_t)(32 * wq) << 16, t_s = tmem + 128 * t + lanes, t_o = t_out + 128 * t + lanes;
        constexpr uint32_t exponent = Half<T>::type == F3M_TYPE_BF16 ? 0x7f80u : 0x7c00u;
        const bool wide = p.wide;
        int tile = 0, cleared = 0, had_b = -1, had_i0 = 0;   // tiles of keys so far, those that were seen in part; the tree that is at hand
        for (int parts = 0;; parts++) {
            // whether there is a part is one thread's word to all: they meet at barriers inside
            const int slot_r = parts % PG_RING;
            if (warp == 0) {
                wait(b_part + 8 * slot_r, (parts / PG_RING) & 1);
                if (lane == 0) go_s[parts & 1] = !gave_up_s && ring_s[slot_r].j1 > 0;
            }
            tc::bar_sync(1, ROWS);
            if (!go_s[parts & 1]) break;
            const PagedPart &part = ring_s[slot_r];
            const PagedItem &w = part.w;   // stays where it is: few of its numbers are worth a register
            const int j0 = part.j0, j1 = part.j1, length = w.length, tokens = w.tokens;
            if (a.parents && (w.b != had_b || w.i0 != had_i0)) {   // depths of the item's tokens, and which new tokens each sees
                had_b = w.b; had_i0 = w.i0;
                for (int m = tid; m < had_i0 + tokens; m += ROWS) parent_s[m] = (int16_t)parent_of(a.parents + w.row0, m);
                tc::bar_sync(1, ROWS);
                if (tid < tokens) {
                    int depth = -1;
                    for (int m = had_i0 + tid; m >= 0; m = parent_s[m]) depth++;
                    depth_s[tid] = (int16_t)depth;
                    for (int k = 0; k < PG_WORDS; k++) above_s[tid][k] = 0u;
                    int d = depth;
                    for (int m = had_i0 + tid; m >= 0; m = parent_s[m], d--)
                        if (depth - d < a.window || length + d < a.sinks) above_s[tid][m >> 5] |= 1u << (m & 31);
                }
                tc::bar_sync(1, ROWS);
            }
            const int token = t * p.tokens + in;   // of the item
            const bool row = in < p.tokens && token < tokens, some = __any_sync(0xffffffffu, row);
            const int pos = length + (a.parents ? (row ? depth_s[token] : 0) : w.i0 + token), up = row ? (a.parents ? length - 1 : pos) : -1;
            const uint32_t *above = a.parents && row ? above_s[token] : nullptr;
            float top = -INFINITY, sum = 0.f;
            uint32_t bad = 0;    // tiles with a seen value that is not finite and was taken out
            for (int j = j0; j < j1; j++, tile++) {
                const int key = w.key(j);
                const bool by_all = seen_by_all(a, w, key);
                wait(b_s + 8 * t, tile & 1);
                __syncwarp();
                tc::fence_after_sync();
                const uint32_t there = there_s[tile % PG_THERE];
                bool whole = by_all && there == 0xffffu;   // then: for this warp's rows
                uint32_t seen[4] = {};
                if (!whole) {
                    // Values that are not finite leave the tile, by the first tile of rows' threads, which may be a tile of keys ahead of the second's.  Scores of this tile tell
                    // that the values in this slot before have landed: the wait names a phase's parity only
                    uint32_t *bads = bad_s[cleared & 1];
                    const uint32_t b_this = b_clear + 8 * (cleared & 1), turn = cleared++ >> 1 & 1;
                    if (t == 0) {
                        const int xv = 2 * tile + 1, sv = xv % slots;
                        wait(b_full + 8 * sv, (xv / slots) & 1);
                        bool finite = true;
                        auto chunk = [&](int c, uint32_t (&v)[4]) {
                            const uint32_t at = slot_tile(sv) + (c >> 3) * PG_BLOCK + tc::swz(r, c & 7);
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
                            return at;
                        };
#pragma unroll 4
                        for (int c = 0; c < 8 * NB; c++) {
                            uint32_t v[4];
                            chunk(c, v);
#pragma unroll
                            for (int k = 0; k < 4; k++) finite &= finite16(v[k], exponent) && finite16(v[k] >> 16, exponent);
                        }
                        if (!finite) {
#pragma unroll 1
                            for (int c = 0; c < 8 * NB; c++) {
                                uint32_t v[4];
                                const uint32_t at = chunk(c, v);
#pragma unroll
                                for (int k = 0; k < 4; k++) v[k] &= (finite16(v[k], exponent) ? 0xffffu : 0u) | (finite16(v[k] >> 16, exponent) ? 0xffff0000u : 0u);
                                sts16(at, v);
                            }
                            tc::fence_async_smem();
                        }
                        const uint32_t b = __ballot_sync(0xffffffffu, !finite);
                        if (lane == 0) {
                            bads[wq] = b;
                            tc::mbar_arrive(b_this);
                        }
                    }
                    wait(b_this, turn);
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        seen[q] = seen_keys(a, length, key + 32 * q, there >> 4 * q, pos, up, above);
                        if (seen[q] & bads[q]) bad |= 1u << ((j - j0) >> tile_shift(part));
                    }
                    whole = __all_sync(0xffffffffu, (seen[0] & seen[1] & seen[2] & seen[3]) == 0xffffffffu);
                }
                if (!some) {   // a warp without rows
                    tc::fence_before_sync();
                    tc::mbar_arrive(b_p + 8 * t);
                    tc::mbar_arrive(b_p2 + 8 * t);
                    continue;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                uint32_t x[2][32];
                tc::tmem_ld32(t_s, x[0]);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    tc::tmem_ld_wait(x[q & 1]);
                    if (q < 3) tc::tmem_ld32(t_s + 32 * (q + 1), x[(q + 1) & 1]);
                    if (whole) {
#pragma unroll
                        for (int c = 0; c < 32; c++) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(x[q & 1][c]));
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c++) mx[c & 3] = fmaxf(mx[c & 3], seen[q] >> c & 1 ? __uint_as_float(x[q & 1][c]) : -INFINITY);
                    }
                }
                tc::tmem_ld32(t_s, x[0]);   // again
                const float high = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                const bool rise = (high - top) * p.c > 8.f;   // also from -inf; not from -inf to -inf
                if (__any_sync(0xffffffffu, rise)) {
                    const float f = rise ? ex2_approx((top - high) * p.c) : 1.f;
                    if (rise) { top = high; sum = sum < PG_NO_SUM ? sum * f : NAN; }
                    if (j > j0)
                        for (int q = 0; q < 2 * NB; q++) {
                            uint32_t o[32];
                            tc::tmem_ld32(t_o + 32 * q, o);
                            tc::tmem_ld_wait(o);
#pragma unroll
                            for (int c = 0; c < 32; c++) o[c] = __float_as_uint(f * __uint_as_float(o[c]));
                            tc::tmem_st32(t_o + 32 * q, o);
                        }
                }
                const float shift = top == -INFINITY ? 0.f : -top * p.c;
                const f32x2 cc = pack2(p.c, p.c), ss = pack2(shift, shift);
                f32x2 add[2] = {pack2(sum, (seen[0] | seen[1] | seen[2] | seen[3]) ? PG_MET : 0.f), pack2(0.f, 0.f)};
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t w16[16];
                    tc::tmem_ld_wait(x[q & 1]);
                    if (q < 3) tc::tmem_ld32(t_s + 32 * (q + 1), x[(q + 1) & 1]);
                    uint32_t(&y)[32] = x[q & 1];
                    if (whole) {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float lo, hi;
                            const f32x2 e = fma2(pack2(__uint_as_float(y[c]), __uint_as_float(y[c + 1])), cc, ss);
                            if (c % 8 == 6) exp2_poly<false>(e, lo, hi);
                            else {
                                unpack2(e, lo, hi);
                                lo = ex2_approx(lo);
                                hi = ex2_approx(hi);
                            }
                            add[(c >> 1) & 1] = add2(add[(c >> 1) & 1], pack2(lo, hi));
                            w16[c >> 1] = Half<T>::pack(lo, hi);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float lo, hi;
                            unpack2(fma2(pack2(__uint_as_float(y[c]), __uint_as_float(y[c + 1])), cc, ss), lo, hi);
                            lo = seen[q] >> c & 1 ? ex2_approx(lo) : 0.f;
                            hi = seen[q] >> (c + 1) & 1 ? ex2_approx(hi) : 0.f;
                            add[(c >> 1) & 1] = add2(add[(c >> 1) & 1], pack2(lo, hi));
                            w16[c >> 1] = Half<T>::pack(lo, hi);
                        }
                    }
                    tc::tmem_st16(t_s + 16 * q, w16);   // over scores that have been read
                    if (q & 1) {
                        tc::tmem_st_wait();
                        tc::fence_before_sync();
                        tc::mbar_arrive((q == 1 ? b_p : b_p2) + 8 * t);
                    }
                }
                float u, v;
                unpack2(add2(add[0], add[1]), u, v);
                sum = u + v;
            }
            const bool cut = part.slot >= 0;
            if (!(sum < PG_NO_SUM) || top == INFINITY) sum = NAN;
            else if (top == -INFINITY && sum != 0.f) sum = cut ? PG_ALL_LOW : NAN;   // 0 / 0, unless another part has more
            const float inv = cut ? 1.f : sum != 0.f ? 1.f / sum : 0.f;   // nothing seen: 0
            const int64_t place = cut ? (int64_t)part.slot * p.rows + token * p.group + head : 0;
            uint16_t *out = reinterpret_cast<uint16_t *>(a.out.data) + (int64_t)(w.row0 + w.i0 + token) * a.out.token_stride + (int64_t)(w.kv_head * p.group + head) * a.out.head_stride;
            float *part_row = p.sums + place * a.c.width;
            wait(b_o + 8 * t, parts & 1);
            __syncwarp();
            tc::fence_after_sync();
            if (some)
#pragma unroll 1
                for (int c = 0; c < 64 * NB; c += 32) {
                    uint32_t o[32];
                    __syncwarp();
                    tc::tmem_ld32(t_o + c, o);
                    tc::tmem_ld_wait(o);
                    if (!row) continue;
                    if (cut) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            if (c + k < a.c.width) *reinterpret_cast<uint4 *>(part_row + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    } else {
                        uint32_t y[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) y[k] = Half<T>::pack(inv * __uint_as_float(o[2 * k]), inv * __uint_as_float(o[2 * k + 1]));
                        store_row32(out, y, c, a.c.width, wide);
                    }
                }
            tc::fence_before_sync();
            tc::mbar_arrive(b_o_read);
            if (row) {
                if (cut) p.stat[place] = make_float2(top * p.c, sum);
                if (bad) {
                    if (cut) poison_row<T>(p, part, bad, pos, up, above, part_row);
                    else poison_row<T>(p, part, bad, pos, up, above, out);
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(b_part_free + 8 * slot_r);
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == COPY) tc::tmem_dealloc(tmem, 256 * TILES);
}

// Items that were cut: a warp a row, 4 columns a lane.  Parts lie in the CTAs from this one on, scaled here to their common maximum, in their order; one that has seen nothing has a sum of 0,
// one whose scores are all -inf weighs nothing beside others, and alone makes the row not a number.
template <typename T>
__global__ void __launch_bounds__(256) paged_join(const __grid_constant__ PagedKernel p) {
    const PagedSplit s = p.split[blockIdx.x];
    const int row = 8 * blockIdx.y + (threadIdx.x >> 5), lane = threadIdx.x & 31, c = 4 * lane;
    if (s.parts == 0 || row >= s.w.tokens * p.group) return;
    auto place = [&](int i) { return (int64_t)(2 * ((int)blockIdx.x + i) + (i == 0)) * p.rows + row; };
    float high = -INFINITY, total = 0.f, o[4] = {};
    bool met = false;
    for (int i = lane; i < s.parts; i += 32) high = fmaxf(high, p.stat[place(i)].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
    if (c >= p.a.c.width) return;
    for (int i = 0; i < s.parts; i++) {
        const float2 t = p.stat[place(i)];
        if (t.y == 0.f) continue;
        met = true;
        const float f = t.y == PG_ALL_LOW ? 0.f : ex2_approx(t.x - high);
        const float4 x = *reinterpret_cast<const float4 *>(p.sums + place(i) * p.a.c.width + c);
        total = fmaf(f, t.y, total);
        o[0] = fmaf(f, x.x, o[0]); o[1] = fmaf(f, x.y, o[1]); o[2] = fmaf(f, x.z, o[2]); o[3] = fmaf(f, x.w, o[3]);
    }
    const float inv = total != 0.f ? 1.f / total : met ? NAN : 0.f;
    uint16_t *out = reinterpret_cast<uint16_t *>(p.a.out.data) + (int64_t)(s.w.row0 + s.w.i0 + row / p.group) * p.a.out.token_stride + (int64_t)(s.w.kv_head * p.group + row % p.group) * p.a.out.head_stride;
    *reinterpret_cast<uint2 *>(out + c) = make_uint2(Half<T>::pack(o[0] * inv, o[1] * inv), Half<T>::pack(o[2] * inv, o[3] * inv));
}

// One launch's share of the workspace: the cut items, their parts' sums and statistics
struct PagedGrid {
    int group, tokens, subs, ctas, rows, q_rows;
    int64_t entries;
    bool used;
    size_t split_bytes() const { return (ctas * sizeof(PagedSplit) + 15) / 16 * 16; }
    size_t bytes(int width) const { return used ? split_bytes() + 2 * (size_t)ctas * rows * (width + 2) * sizeof(float) : 0; }
};
static PagedGrid paged_grid(const f3m_seqs &s, const f3m_cache &c, int heads, int tiles) {
    PagedGrid g;
    g.group = heads / c.kv_heads;
    g.tokens = SEQ_TILE / g.group;
    g.subs = (std::min(s.longest, 2 * SEQ_TILE) + 2 * g.tokens - 1) / (2 * g.tokens);
    g.entries = (int64_t)s.pairs * g.subs;
    const int64_t most = ((int64_t)c.table_pages * c.page_tokens + s.longest) / SEQ_TILE + 1, sms = NUM_SMS_HINT * (3 - tiles);   // tiles of keys of an item; CTAs that run at a time
    g.ctas = (int)std::min(sms, std::min(g.entries * c.kv_heads, sms) * most);
    g.q_rows = (std::min(s.longest, g.tokens) * g.group + 7) / 8 * 8;
    g.rows = (std::min(s.longest, tiles * g.tokens) * g.group + 1) / 2 * 2;
    // more tokens than a tile of rows holds make items of two; whether one is left of one tile is known of a single sequence
    auto odd = [&](int n) { const int left = n % (2 * g.tokens); return left > 0 && left <= g.tokens; };
    g.used = tiles == 2 ? s.longest > g.tokens : s.sequences > 1 || odd(s.longest % (2 * SEQ_TILE)) || (s.longest >= 2 * SEQ_TILE && odd(2 * SEQ_TILE));
    return g;
}
size_t paged_workspace(const f3m_seqs &s, const f3m_cache &c, int heads) {
    if (heads / c.kv_heads > SEQ_TILE) return 0;
    return paged_grid(s, c, heads, 1).bytes(c.width) + paged_grid(s, c, heads, 2).bytes(c.width);
}

template <typename T, int NB, int TILES>
static void paged_launch(PagedKernel &p, const PagedGrid &g, void *ws, cudaStream_t s) {
    // what half an SM holds, or a whole one, beside what is static (2 KB) and what the system takes of each CTA (1 KB)
    constexpr int room = (TILES == 1 ? 233472 / 2 : 233472) - 1024 - 2048, slot = NB * PG_BLOCK;
    p.q_rows = TILES == 1 ? g.q_rows : SEQ_TILE;
    const int fixed = 1024 + 128 * TILES * PG_WORDS * 4, rows = NB * p.q_rows * 128;
    // a second place for rows where it takes none of the keys': the next item's are there in time
    p.slots = (room - fixed - TILES * rows) / slot;
    p.places = TILES == 2 || p.slots == (room - fixed - 2 * rows) / slot ? 2 : 1;
    p.slots = std::min(p.slots, PG_MAX_SLOTS);
    const int bytes = fixed + p.places * rows + p.slots * slot;
    p.rows = g.rows;
    p.split = reinterpret_cast<PagedSplit *>(ws);
    p.sums = reinterpret_cast<float *>(reinterpret_cast<char *>(ws) + g.split_bytes());
    p.stat = reinterpret_cast<float2 *>(p.sums + 2 * (size_t)g.ctas * g.rows * p.a.c.width);
    auto kernel = paged_tiles<T, NB, TILES>;
    static SharedMemory allowed;
    allowed.allow(kernel, room);
    kernel<<<g.ctas, 128 * TILES + 64, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
    paged_join<T><<<dim3(g.ctas, (g.rows + 7) / 8), 256, 0, s>>>(p);
    F3M_LAUNCH_CHECK();
}

template <typename T>
static void paged_t(const PagedArgs &a, cudaStream_t s) {
    PagedKernel p;
    p.a = a;
    const PagedGrid one = paged_grid(a.s, a.c, a.heads, 1), two = paged_grid(a.s, a.c, a.heads, 2);
    F3M_REQUIRE(one.entries <= 0x7fffffff - 512, F3M_ERR_OVERFLOW, "%lld tiles of new tokens do not fit in 31 bits", (long long)one.entries);
    const int top = (int)std::min<int64_t>((int64_t)a.c.table_pages * a.c.page_tokens + a.s.longest, 0x7fffff00);   // no position is beyond
    p.a.window = std::min(a.window, std::max(top, 1));
    p.a.sinks = std::min(a.sinks, top);
    p.group = one.group; p.tokens = one.tokens; p.subs = one.subs; p.entries = (int)one.entries;
    p.page_shift = 31 - __builtin_clz(a.c.page_tokens);
    p.box = std::min(a.c.page_tokens, SEQ_TILE);
    p.wide = rows_wide(a.out);
    p.c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 0x1p-149f);   // a scale of zero: all weights are one, whatever finite number the scores are
    p.err = seq_error_word();
    f3m_cache c = a.c;
    if (c.pages == 0) {   // no page is read: the maps need an address
        c.pages = 1;
        c.k = c.v = f3m_pages{a.q.data, c.width, c.width, c.width};
    }
    p.mk = page_tensor_map(Half<T>::type, c, c.k, p.box);
    p.mv = page_tensor_map(Half<T>::type, c, c.v, p.box);
    // copies of a tile of rows bring whole tokens, no more than the longest sequence has
    const int tokens = std::min(one.tokens, a.s.longest);
    p.q_box = tokens * one.group;
    p.mq = seq_tensor_map(Half<T>::type, a.q, a.s.tokens, a.heads, a.c.width, one.group, tokens);
    char *ws = reinterpret_cast<char *>(a.ws);
    if (two.used) a.c.width <= 64 ? paged_launch<T, 1, 2>(p, two, ws + one.bytes(a.c.width), s) : paged_launch<T, 2, 2>(p, two, ws + one.bytes(a.c.width), s);
    if (one.used) a.c.width <= 64 ? paged_launch<T, 1, 1>(p, one, ws, s) : paged_launch<T, 2, 1>(p, one, ws, s);
}

void paged_attention(int type, const PagedArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? paged_t<__nv_bfloat16>(a, s) : paged_t<__half>(a, s); }

// ---- accepted paths -----------------------------------------------------------------------------------------------------------
// A CTA has the keys or the values of one head of a sequence, and takes its places in order, KP_ROWS at a time: read, then written.  A place is read for one in front of it or
// for itself (kept[j] >= j), so that what is written has been read.  64 paths of up to 30 tokens, 8 heads, width 128: three dependent loads and a store, 6.2 us (a thread for all
// places of 16 bytes, 8 at a time: 17.9 in all).
constexpr int KP_STEP = 16, KP_EACH = 4, KP_ROWS = KP_STEP * KP_EACH, KP_THREADS = 16 * KP_STEP;
__global__ void __launch_bounds__(KP_THREADS) keep_paths(const __grid_constant__ f3m_cache c, const int *kept, int64_t kept_stride, int most, const int *counts) {
    const int b = blockIdx.x, h = blockIdx.y >> 1, col = 8 * (threadIdx.x & 15), length = paged_length(c, b), count = min(max(counts[b], 0), most);
    const f3m_pages &p = blockIdx.y & 1 ? c.v : c.k;
    uint16_t *data = reinterpret_cast<uint16_t *>(p.data) + col;
    for (int j0 = 0; j0 < count; j0 += KP_ROWS) {
        uint4 v[KP_EACH];
        int64_t to[KP_EACH];
#pragma unroll
        for (int r = 0; r < KP_EACH; r++) {
            const int j = j0 + KP_STEP * r + (threadIdx.x >> 4), m = j < count && col < c.width ? kept[b * kept_stride + j] : -1;
            to[r] = -1;
            if (m <= j) continue;   // its place already, or no place of a path
            const int page = paged_page(c, b, (int64_t)length + m), there = paged_page(c, b, (int64_t)length + j);
            if (page < 0 || there < 0) continue;
            to[r] = paged_at(c, p, there, (int64_t)length + j, h);
            v[r] = *reinterpret_cast<const uint4 *>(data + paged_at(c, p, page, (int64_t)length + m, h));
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < KP_EACH; r++)
            if (to[r] >= 0) *reinterpret_cast<uint4 *>(data + to[r]) = v[r];
        __syncthreads();
    }
}

void paged_keep(const f3m_cache &c, const int *kept, int64_t kept_stride, int most, const int *counts, cudaStream_t s) {
    F3M_REQUIRE(c.kv_heads <= 32767, F3M_ERR_UNSUPPORTED, "%d key heads", c.kv_heads);
    keep_paths<<<dim3(c.sequences, 2 * c.kv_heads), KP_THREADS, 0, s>>>(c, kept, kept_stride, most, counts);
    F3M_LAUNCH_CHECK();
}

}  // namespace f3m
