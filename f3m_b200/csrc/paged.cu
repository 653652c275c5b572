// A cache of keys and values in pages: new tokens appended, their attention over it, accepted paths of drafted trees.
#include <algorithm>
#include "seq.cuh"

namespace f3m {

// ---- new tokens to their pages ----------------------------------------------------------------------------------------------
// A CTA has AP_TOKENS neighbouring tokens of a sequence.  Their places and angles are taken once for all heads: the part of a whole turn is position * turns modulo
// 2^64, exact for any position, and what is left, in FP32, is at most half a turn.  Then 16-byte vectors, as (token, head, vector); a vector of a half-split
// rotation brings its partner.  Memory is the bound: every array is read and written once.
constexpr int AP_TOKENS = 4, AP_THREADS = 256;

template <typename T>
__device__ __forceinline__ void rotate8(uint4 &x, uint4 &y, const float2 *turn, bool interleaved) {
    uint32_t *xs = reinterpret_cast<uint32_t *>(&x), *ys = reinterpret_cast<uint32_t *>(&y);
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = Half<T>::unpack(xs[i]), c = turn[i];
            xs[i] = Half<T>::pack(f.x * c.x - f.y * c.y, f.x * c.y + f.y * c.x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = Half<T>::unpack(xs[i]), g = Half<T>::unpack(ys[i]), c = turn[2 * i], d = turn[2 * i + 1];
            xs[i] = Half<T>::pack(f.x * c.x - g.x * c.y, f.y * d.x - g.y * d.y);
            ys[i] = Half<T>::pack(f.x * c.y + g.x * c.x, f.y * d.y + g.y * d.x);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(AP_THREADS) append_tokens(const __grid_constant__ AppendArgs a) {
    __shared__ int slot_s[AP_TOKENS], pos_s[AP_TOKENS], page_s[AP_TOKENS];
    __shared__ float2 turn_s[AP_TOKENS][F3M_MAX_WIDTH / 2];
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, blockIdx.x)];
    const int i0 = e.z + AP_TOKENS * blockIdx.y, m = min(AP_TOKENS, min(e.z + SEQ_TILE, e.y) - i0), half = a.rotation.columns / 2;
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
        turn_s[t][i] = make_float2(c, s);
    }
    __syncthreads();
    const int vectors = a.c.width / 8, moved = a.rotation.interleaved ? 0 : half / 8;   // the second half's vectors come with the first's
    const int turned = vectors - moved, rows = a.heads + a.c.kv_heads, units = rows * turned + a.c.kv_heads * vectors;
    for (int x = threadIdx.x; x < m * units; x += AP_THREADS) {
        const int t = x / units, u = x % units;
        const bool value = u >= rows * turned;
        const int w = value ? u - rows * turned : u, per = value ? vectors : turned;
        int h = w / per, c = w % per;
        const bool query = !value && h < a.heads;
        if (!value && !query) h -= a.heads;
        const bool pair = !value && c < moved, rotated = !value && 8 * c < (moved ? half : 2 * half);
        if (!value && c >= moved) c += moved;   // behind the pairs; of no consequence where moved is 0
        const f3m_rows &from = query ? a.q : value ? a.v : a.k;
        const uint16_t *src = reinterpret_cast<const uint16_t *>(from.data) + (int64_t)(e.x + i0 + t) * from.token_stride + (int64_t)h * from.head_stride + 8 * c;
        uint16_t *dst;
        if (query) dst = reinterpret_cast<uint16_t *>(a.q_out.data) + (int64_t)(e.x + i0 + t) * a.q_out.token_stride + (int64_t)h * a.q_out.head_stride + 8 * c;
        else {
            if (page_s[t] < 0) continue;
            const f3m_pages &p = value ? a.c.v : a.c.k;
            dst = reinterpret_cast<uint16_t *>(p.data) + paged_at(a.c, p, page_s[t], slot_s[t], h) + 8 * c;
        }
        uint4 f = *reinterpret_cast<const uint4 *>(src), g = make_uint4(0u, 0u, 0u, 0u);
        if (pair) g = *reinterpret_cast<const uint4 *>(src + half);
        if (rotated) rotate8<T>(f, g, turn_s[t] + (a.rotation.interleaved ? 4 * c : 8 * c), a.rotation.interleaved);
        *reinterpret_cast<uint4 *>(dst) = f;
        if (pair) *reinterpret_cast<uint4 *>(dst + half) = g;
    }
}

void paged_append(int type, const AppendArgs &a, cudaStream_t s) {
    const dim3 grid(a.s.tiles, (std::min(a.s.longest, SEQ_TILE) + AP_TOKENS - 1) / AP_TOKENS);
    if (type == F3M_TYPE_BF16) append_tokens<__nv_bfloat16><<<grid, AP_THREADS, 0, s>>>(a);
    else append_tokens<__half><<<grid, AP_THREADS, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}

// ---- attention of new tokens ------------------------------------------------------------------------------------------------
// An item is one key head and as many new tokens as make two tiles of 128 rows, (token, head) of the heads that share it; it walks over the tiles of 128
// keys that some of its rows see.  CTAs, one per SM, share all items' tiles evenly: CTA c of G takes tiles c U / G .. (c + 1) U / G of U, cuts through
// items where that falls, and paged_join puts the parts together.  How long a sequence is stands on the device only, so that each CTA counts for itself.
//
// As in window attention S = Q K^T goes to tensor memory, a thread takes the weights of one row and writes them over S, from where they go into O += P V, and two
// streams take turns, one's weights while the other's products run.  The streams are the item's two tiles of rows, or, where it has one only (one token, a
// drafted tree), every other tile of keys: rows of the same lanes, so that at the end each thread adds the two O's itself.
//
// Keys that only a part of the item's rows sees (the window's edge, new tokens, a tree, missing pages) go by bits, a word for 32 of them.  A value that is not finite would
// reach every row there, as zero times it: it is taken out of the tile, and added to the rows that see it when they have been written (poison_row).
constexpr int PG_COPY = 8, PG_PRODUCTS = 9, PG_THREADS = 320, PG_BLOCK = SEQ_TILE * 128, PG_RING = 4, PG_SLOTS = 10, PG_THERE = 8, PG_ITEM = 1;
constexpr float PG_NO_SUM = 0x1p60f;   // some exponent was not a number (exp2_poly)
constexpr int PG_WORDS = F3M_TREE_MAX / 32;

struct PagedItem {
    int row0, n, b, i0, tokens, length;   // the sequence's first row, new tokens, number; first token of the item, how many; tokens in the cache
    int kv_head, tiles_q, sinks, first, keys;   // tiles of rows; tiles of keys: the first `sinks` of the sequence, then those from tile `first` on; `keys` in all
    __device__ __forceinline__ int key(int j) const { return SEQ_TILE * (j < sinks ? j : first + j - sinks); }
    __device__ __forceinline__ int cost() const { return keys ? keys + PG_ITEM : 0; }   // in tiles; what an item takes beside them comes behind its last
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
    int rows;              // of a part's place in the workspace
    bool wide;
    float c;               // |scale| log2(e)
    float2 *stat;          // (2 G, rows): maximum, sum of weights
    float *sums;           // (2 G, rows, width)
    PagedSplit *split;     // (G)
    int *err;
};

// Entry e: a sequence's tokens, without a key head; no tokens: none are left
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
    w.tiles_q = w.tokens > p.tokens ? 2 : 1;
    // the first new token that a row may be, by its position: a tree's may be a root
    w.first = max(0, w.length + (a.parents ? 0 : w.i0) - a.window + 1) / SEQ_TILE;
    w.sinks = min((a.sinks + SEQ_TILE - 1) / SEQ_TILE, w.first);
    w.keys = w.tokens ? w.sinks + (w.length + w.i0 + w.tokens - 1) / SEQ_TILE - w.first + 1 : 0;
    return w;
}
// Whether all rows of the item see all keys of a tile; there: which of its 16 groups of 8 keys have a page
__device__ __forceinline__ bool seen_by_all(const PagedKernel &p, const PagedItem &w, int key, uint32_t there) {
    const PagedArgs &a = p.a;
    const int last = w.length + w.i0 + w.tokens - 1;   // the furthest position
    return there == 0xffffu && key + SEQ_TILE - 1 <= w.length + (a.parents ? -1 : w.i0) && (last - key < a.window || key + SEQ_TILE <= a.sinks);
}
__device__ __forceinline__ uint32_t ones(int from, int to) {   // bits from .. to - 1 of a word
    from = max(from, 0);
    to = min(to, 32);
    return to > from ? (0xffffffffu >> (32 - to + from)) << from : 0u;
}
// The keys from `at` to at + 31 that a row at position pos sees; `there` of their four groups of 8.  up: its last key but for a tree's; above: a tree's new tokens that it sees
__device__ __forceinline__ uint32_t seen_keys(const PagedArgs &a, const PagedItem &w, int at, uint32_t there, int pos, int up, const uint32_t *above) {
    uint32_t m = (ones(pos - a.window + 1 - at, 32) | ones(0, a.sinks - at)) & ones(0, up + 1 - at);
    if (above) {
        const int bit = at - w.length, k = bit >> 5;
        const uint32_t lo = k >= 0 && k < PG_WORDS ? above[k] : 0u, hi = k >= -1 && k + 1 < PG_WORDS ? above[k + 1] : 0u;
        m |= __funnelshift_r(lo, hi, bit & 31);
    }
    const uint32_t groups = (there & 1u) | (there & 2u) << 7 | (there & 4u) << 14 | (there & 8u) << 21;
    return m & groups * 0xffu;
}

__device__ __forceinline__ bool finite16(uint32_t v, uint32_t exponent) { return (v & exponent) != exponent; }   // the lower half of a word

// Values that are not finite, of keys in tiles that were cleared of them, to columns c0 .. c1 - 1 of a row that sees them
template <typename T, typename O>
__device__ __noinline__ void poison_row(const PagedKernel &p, const PagedPart &part, int pos, int up, const uint32_t *above, O *row, int c0, int c1) {
    const PagedArgs &a = p.a;
    const PagedItem &w = part.w;
    for (int j = part.j0; j < part.j1; j++) {
        const int key = w.key(j);
        uint32_t there = 0;
        for (int g = 0; g < SEQ_TILE / 8; g++) there |= (uint32_t)(paged_page(a.c, w.b, (int64_t)key + 8 * g) >= 0) << g;
        if (seen_by_all(p, w, key, there)) continue;
        for (int q = 0; q < 4; q++)
            for (uint32_t m = seen_keys(a, w, key + 32 * q, there >> 4 * q, pos, up, above); m; m &= m - 1) {
                const int64_t slot = key + 32 * q + __ffs(m) - 1;
                const uint16_t *v = reinterpret_cast<const uint16_t *>(a.c.v.data) + paged_at(a.c, a.c.v, paged_page(a.c, w.b, slot), slot, w.kv_head);
                for (int c = c0; c < c1; c++) {
                    const float x = Half<T>::unpack(v[c]).x;
                    if (isfinite(x)) continue;
                    if constexpr (sizeof(O) == 4) row[c] += x;
                    else row[c] = (O)Half<T>::pack(Half<T>::unpack(row[c]).x + x, 0.f);
                }
            }
    }
}

template <typename T, int NB>
__global__ void __launch_bounds__(PG_THREADS, 1) paged_tiles(const __grid_constant__ PagedKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * PG_SLOTS + 2 * PG_RING + 14];
    __shared__ PagedPart ring_s[PG_RING];
    __shared__ long long warp_s[PG_THREADS / 32], start_s[2];
    __shared__ uint32_t tmem_s, bad_s[2][2][4], there_s[PG_THERE];
    __shared__ float2 stat_s[2][SEQ_TILE];
    __shared__ int gave_up_s, go_s[2];
    __shared__ int16_t parent_s[F3M_TREE_MAX], depth_s[F3M_TREE_MAX];
    const PagedArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int slots = NB == 2 ? 4 : 10;
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u;
    auto q_tile = [&](int t) { return smem + t * NB * PG_BLOCK; };
    auto slot_tile = [&](int s) { return smem + (2 + s) * NB * PG_BLOCK; };
    uint32_t(*above_s)[PG_WORDS] = reinterpret_cast<uint32_t(*)[PG_WORDS]>(raw + (smem - tc::smem_u32(raw)) + (2 + slots) * NB * PG_BLOCK);

    if (warp == PG_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = b_full + 8 * PG_SLOTS, b_part = b_free + 8 * PG_SLOTS, b_part_free = b_part + 8 * PG_RING, b_q = b_part_free + 8 * PG_RING,
                   b_q_free = b_q + 16, b_s = b_q + 32, b_p = b_q + 48, b_p2 = b_q + 64, b_o = b_q + 80, b_o_read = b_q + 96, b_none = b_q + 104;
    if (tid == 0) {
        for (int i = 0; i < 2 * PG_SLOTS; i++) tc::mbar_init(b_full + 8 * i, 1);       // landed, free
        for (int i = 0; i < PG_RING; i++) {
            tc::mbar_init(b_part + 8 * i, 1);                                          // a part is told
            tc::mbar_init(b_part_free + 8 * i, 9);                                     // and done with, by nine warps
        }
        for (int t = 0; t < 2; t++) {
            tc::mbar_init(b_q + 8 * t, 1);       // a tile of rows landed, free
            tc::mbar_init(b_q_free + 8 * t, 1);
            tc::mbar_init(b_s + 8 * t, 1);       // S ready
            tc::mbar_init(b_p + 8 * t, 128);     // weights of the first 64 keys written
            tc::mbar_init(b_p2 + 8 * t, 128);    // of the other 64
            tc::mbar_init(b_o + 8 * t, 1);       // O ready
        }
        tc::mbar_init(b_o_read, 256);            // both read
        tc::mbar_init(b_none, 1);                // no products in flight
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    // tiles of all items, and where this CTA's begin
    auto tiles_of = [&](int e) { return e < p.entries ? (long long)paged_item(p, e).cost() * a.c.kv_heads : 0ll; };
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
        for (int i = 0; i < PG_THREADS / 32; i++) {
            if (i == warp) before = all;
            all += warp_s[i];
        }
        return v + before;
    };
    long long total = 0, mine = 0, up_to = 0, sum;
    for (int e = 0; e < p.entries; e += PG_THREADS) {
        mine = tiles_of(e + tid);
        up_to = scan(mine, sum);
        total += sum;
    }
    const int ctas = (int)min((long long)gridDim.x, total), cta = blockIdx.x;   // a tile at least for each
    const long long u0 = cta < ctas ? cta * total / ctas : total, u1 = cta < ctas ? (cta + 1) * total / ctas : total;
    long long base = 0;
    for (int e = 0; e < p.entries; e += PG_THREADS) {
        if (p.entries > PG_THREADS) {
            mine = tiles_of(e + tid);
            up_to = scan(mine, sum);
        }
        if (u0 < base + up_to && u0 >= base + up_to - mine) { start_s[0] = e + tid; start_s[1] = u0 - (base + up_to - mine); }
        base += sum;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s;

    if (warp == PG_COPY) {
        // ---- parts told to the others, copies; a lane has a page of a tile ----
        // Copies of a part come in the order K0 K1 V0 K2 V1 .., without a stop between parts: values are wanted a tile's weights later than keys, and would only hold their place.
        int x = 0, y = 0, parts = 0, e = u0 < u1 ? (int)start_s[0] : 0, e0 = e, uses0 = 0, uses1 = 0, turn = 0;   // copies, tiles, parts so far; uses of the places for rows
        long long left = u1 - u0;
        bool stop = false;   // of the whole warp
        const int boxes = SEQ_TILE / p.box;
        const uint32_t page_mask = (1u << p.page_shift) - 1;
        auto wait_all = [&](uint32_t bar, uint32_t parity) {
            wait(bar, parity);
            stop = __any_sync(0xffffffffu, gave_up_s);
        };
        // entries are read 32 at a time, a lane each
        PagedItem held = paged_item(p, min(e + lane, p.entries - 1)), w;
        auto entry = [&](int i) {
            if (i - e0 >= 32) {
                e0 = i;
                held = paged_item(p, min(i + lane, p.entries - 1));
            }
            PagedItem z;
#define F3M_SAME(m) z.m = __shfl_sync(0xffffffffu, held.m, i - e0)
            F3M_SAME(row0); F3M_SAME(n); F3M_SAME(b); F3M_SAME(i0); F3M_SAME(tokens); F3M_SAME(length); F3M_SAME(kv_head); F3M_SAME(tiles_q); F3M_SAME(sinks); F3M_SAME(first); F3M_SAME(keys);
#undef F3M_SAME
            return z;
        };
        auto rows_of = [&](int place, const PagedItem &z, int tile) {
            int &uses = place ? uses1 : uses0;
            if (uses && !stop) wait_all(b_q_free + 8 * place, (uses - 1) & 1);
            if (stop) return;
            if (lane == 0) {
                tc::mbar_expect_tx(b_q + 8 * place, NB * p.tokens * p.group * 128);
                for (int c = 0; c < NB; c++)
                    tc::tma_rows(q_tile(place) + c * PG_BLOCK, &p.mq, 64 * c, z.kv_head * p.group, z.row0 + z.i0 + tile * p.tokens, b_q + 8 * place);
            }
            uses++;
        };
        auto page_at = [&](const PagedItem &z, int k) { return lane < boxes ? paged_page(a.c, z.b, (int64_t)z.key(k) + lane * p.box) : -1; };
        w = entry(e);
        int j = 0;
        if (left) { w.kv_head = min((int)(start_s[1] / w.cost()), a.c.kv_heads - 1); j = (int)(start_s[1] % w.cost()); }
        if (lane == 0) p.split[cta].parts = 0;
        auto next = [&] {   // the item behind this one
            left -= min(left, (long long)w.cost() - j);
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
            const PagedItem now = w;
            PagedPart t{now, j, (int)min((long long)now.keys, j + left), -1};
            if (t.j0 > 0 || t.j1 < now.keys) t.slot = 2 * cta + (t.j0 == 0);
            if (t.j0 == 0 && t.j1 < now.keys) {   // the item's last tile is keys - j1 behind this CTA's
                const long long u = u1 - 1 + now.keys - t.j1;
                if (lane == 0) p.split[cta] = {now, (int)(((u + 1) * ctas - 1) / total) - cta + 1};
            }
            const int r = parts % PG_RING;
            if (parts >= PG_RING) wait_all(b_part_free + 8 * r, (parts / PG_RING - 1) & 1);
            if (stop) break;
            if (lane == 0) {
                ring_s[r] = t;
                tc::mbar_arrive(b_part + 8 * r);
            }
            parts++;
            next();
            const int later = left ? page_at(w, 0) : -1;   // of the next part, whose copies are to follow without a stop
            if (now.tiles_q == 2) {
                rows_of(0, now, 0);
                rows_of(1, now, 1);
            } else {
                rows_of(turn, now, 0);
                turn ^= 1;
            }
            const int all = t.j1 - t.j0;
            int even = -1, odd = -1, ahead = page;   // pages of the last tiles of keys, of the next
            for (int i = 0; i < 2 * all && !stop; i++, x++) {
                const bool values = i && (i % 2 == 0 || (i + 1) / 2 == all);
                const int k = !values ? (i + 1) / 2 : i % 2 ? all - 1 : i / 2 - 1, s = x % slots, row = (int)((uint32_t)(now.key(t.j0 + k) + lane * p.box) & page_mask);
                uint32_t there = 0;
                if (!values) {
                    (k & 1 ? odd : even) = ahead;
                    there = __ballot_sync(0xffffffffu, ahead >= 0);
                    there = __ballot_sync(0xffffffffu, lane < SEQ_TILE / 8 && there >> (8 * lane / p.box) & 1u);   // of 16 groups of 8 keys
                    ahead = k + 1 < all ? page_at(now, t.j0 + k + 1) : -1;
                }
                if (x >= slots) wait_all(b_free + 8 * s, (x / slots - 1) & 1);
                if (stop) break;
                if (lane == 0) {
                    if (!values) there_s[(y + k) % PG_THERE] = there;
                    tc::mbar_expect_tx(b_full + 8 * s, NB * PG_BLOCK);
                }
                __syncwarp();
                if (lane < boxes)   // of a page that is not there zeros come
                    for (int c = 0; c < NB; c++)
                        tc::tma_page(slot_tile(s) + c * PG_BLOCK + lane * p.box * 128, values ? &p.mv : &p.mk, 64 * c, now.kv_head, row, k & 1 ? odd : even, b_full + 8 * s);
            }
            y += all;
            page = later;
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
            if (uses0) wait.drain(b_q, (uses0 - 1) & 1);
            if (uses1) wait.drain(b_q + 8, (uses1 - 1) & 1);
        }
    } else if (warp == PG_PRODUCTS) {
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        // a negative scale turns S's sign: bit 13 negates A
        const uint32_t i_s = tc::idesc_f16(bf, 128, 128, false, false) | (a.scale < 0.f ? 1u << 13 : 0u), i_o = tc::idesc_f16(bf, 128, 64 * NB, false, true);
        int x = 0, np[2] = {0, 0}, uses[2] = {0, 0}, turn = 0;
        for (int parts = 0;; parts++) {
            const int r = parts % PG_RING;
            wait(b_part + 8 * r, (parts / PG_RING) & 1);
            if (__any_sync(0xffffffffu, gave_up_s)) break;
            const PagedPart &part = ring_s[r];
            const int tiles_q = part.w.tiles_q, keys = part.j1 - part.j0, end = part.j1;
            __syncwarp();
            if (end == 0) break;
            if (lane == 0) tc::mbar_arrive(b_part_free + 8 * r);
            const bool by_keys = tiles_q == 1;
            const int ahead = by_keys ? 2 : 1;   // a stream's next tile of keys
            auto keys_at = [&](int k) { return x + (k ? 2 * k - 1 : 0); };
            auto values_at = [&](int k) { return x + min(2 * k + 2, 2 * keys - 1); };
            auto scores = [&](int t, int k) {
                const int at = keys_at(k), s = at % slots, place = by_keys ? turn : t;
                wait(b_full + 8 * s, (at / slots) & 1);
                tc::fence_after_sync();
                if (tc::elect()) {
                    tc::product_rows<NB>(tmem + 128 * t, q_tile(place), slot_tile(s), i_s);
                    tc::mma_commit(b_s + 8 * t);
                    if (by_keys || t == 1) tc::mma_commit(b_free + 8 * s);
                    if (k == keys - 1) tc::mma_commit(b_q_free + 8 * place);
                }
            };
            for (int t = 0; t < 2; t++)
                if (!by_keys || t == turn) wait(b_q + 8 * t, uses[t]++ & 1);
            scores(0, 0);
            if (!by_keys) scores(1, 0);
            else if (keys > 1) scores(1, 1);
            if (parts) wait(b_o_read, (parts - 1) & 1);
            for (int k = 0; k < keys; k++) {
                const int at = values_at(k), sv = at % slots;
                wait(b_full + 8 * sv, (at / slots) & 1);
                for (int i = 0; i < tiles_q; i++) {
                    const int t = by_keys ? k & 1 : i;
                    const bool begun = k >= ahead, more = k + ahead < keys;
                    wait(b_p + 8 * t, np[t] & 1);
                    tc::fence_after_sync();
                    if (tc::elect()) tc::product_tmem64(tmem + 256 + 128 * t, tmem + 128 * t, slot_tile(sv), i_o, begun);
                    wait(b_p2 + 8 * t, np[t] & 1);
                    np[t]++;
                    tc::fence_after_sync();
                    if (tc::elect()) {
                        tc::product_tmem64(tmem + 256 + 128 * t, tmem + 128 * t + 32, slot_tile(sv) + 64 * 128, i_o, 1);
                        if (i == tiles_q - 1) tc::mma_commit(b_free + 8 * sv);
                        if (!more) tc::mma_commit(b_o + 8 * t);
                    }
                    if (more) scores(t, k + ahead);
                }
            }
            x += 2 * keys;
            if (by_keys) turn ^= 1;
        }
        wait.drain_products(b_none);
    } else {
        // ---- weights: thread r of a stream has row r of its tile ----
        const int t = warp >> 2, r = tid & 127, wq = warp & 3, in = r / p.group, head = r % p.group;
        const uint32_t lanes = (uint32_t)(32 * wq) << 16, t_s = tmem + 128 * t + lanes, t_o = tmem + 256 + lanes;
        constexpr uint32_t exponent = Half<T>::type == F3M_TYPE_BF16 ? 0x7f80u : 0x7c00u;
        int ns = 0, no[2] = {0, 0}, x0 = 0, had_b = -1, had_i0 = 0;
        for (int parts = 0;; parts++) {
            // whether there is a part is one thread's word to all: they meet at barriers inside
            const int slot_r = parts % PG_RING;
            if (warp == 0) {
                wait(b_part + 8 * slot_r, (parts / PG_RING) & 1);
                if (lane == 0) go_s[parts & 1] = !gave_up_s && ring_s[slot_r].j1 > 0;
            }
            tc::bar_sync(3, 256);
            if (!go_s[parts & 1]) break;
            const PagedPart &part = ring_s[slot_r];
            const PagedItem &w = part.w;   // stays where it is: few of its numbers are worth a register
            const int j0 = part.j0, j1 = part.j1, length = w.length, tokens = w.tokens;
            const bool by_keys = w.tiles_q == 1;
            int scrubs = 0;
            if (a.parents && (w.b != had_b || w.i0 != had_i0)) {   // depths of the item's tokens, and which new tokens each sees
                had_b = w.b; had_i0 = w.i0;
                for (int m = tid; m < had_i0 + tokens; m += 256) parent_s[m] = (int16_t)parent_of(a.parents + w.row0, m);
                tc::bar_sync(3, 256);
                if (tid < tokens) {
                    int depth = -1;
                    for (int m = had_i0 + tid; m >= 0; m = parent_s[m]) depth++;
                    depth_s[tid] = (int16_t)depth;
                    for (int k = 0; k < PG_WORDS; k++) above_s[tid][k] = 0u;
                    int d = depth;
                    for (int m = had_i0 + tid; m >= 0; m = parent_s[m], d--)
                        if (depth - d < a.window || length + d < a.sinks) above_s[tid][m >> 5] |= 1u << (m & 31);
                }
                tc::bar_sync(3, 256);
            }
            const int token = by_keys ? in : t * p.tokens + in;   // of the item
            const bool row = in < p.tokens && token < tokens, some = __any_sync(0xffffffffu, row);
            const int pos = length + (a.parents ? (row ? depth_s[token] : 0) : w.i0 + token), up = row ? (a.parents ? length - 1 : pos) : -1;
            const uint32_t *above = a.parents && row ? above_s[token] : nullptr;
            const int step = by_keys ? 2 : 1, k0 = by_keys ? j0 + t : j0;
            float top = -INFINITY, sum = 0.f;
            bool bad = false;
            for (int j = k0; j < j1; j += step) {
                const int key = w.key(j);
                wait(b_s + 8 * t, ns & 1);
                ns++;
                __syncwarp();
                tc::fence_after_sync();
                const uint32_t there = there_s[(x0 / 2 + j - j0) % PG_THERE];
                const bool whole = seen_by_all(p, w, key, there);
                uint32_t seen[4] = {};
                if (!whole) {
                    // Values that are not finite leave the tile.  Scores of this tile tell that the values in this slot before have landed: the wait names a phase's parity only
                    uint32_t *bads = bad_s[by_keys ? t : 0][scrubs++ & 1];
                    if (by_keys || t == 0) {
                        const int xv = x0 + min(2 * (j - j0) + 2, 2 * (j1 - j0) - 1), sv = xv % slots;
                        wait(b_full + 8 * sv, (xv / slots) & 1);
                        bool finite = true;
                        auto chunk = [&](int c, uint32_t (&v)[4]) {
                            const uint32_t at = slot_tile(sv) + (c >> 3) * PG_BLOCK + tc::swz(r, c & 7);
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
                            return at;
                        };
#pragma unroll
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
                        if (lane == 0) bads[wq] = b;
                    }
                    if (by_keys) tc::bar_sync(1 + t, 128);
                    else tc::bar_sync(3, 256);
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        seen[q] = seen_keys(a, w, key + 32 * q, there >> 4 * q, pos, up, above);
                        bad |= (seen[q] & bads[q]) != 0u;
                    }
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
                    if (j > k0)
                        for (int q = 0; q < 2 * NB; q++) {
                            uint32_t o[32];
                            tc::tmem_ld32(t_o + 128 * t + 32 * q, o);
                            tc::tmem_ld_wait(o);
#pragma unroll
                            for (int c = 0; c < 32; c++) o[c] = __float_as_uint(f * __uint_as_float(o[c]));
                            tc::tmem_st32(t_o + 128 * t + 32 * q, o);
                        }
                }
                const float shift = top == -INFINITY ? 0.f : -top * p.c;
                const f32x2 cc = pack2(p.c, p.c), ss = pack2(shift, shift);
                f32x2 add[2] = {pack2(sum, 0.f), pack2(0.f, 0.f)};
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
            if (!(sum < PG_NO_SUM) || top == INFINITY) sum = NAN;
            // outputs: of a stream's own rows, or half the columns of both streams' sums
            float f[2] = {t == 0 ? 1.f : 0.f, t == 0 ? 0.f : 1.f};
            int c0 = 0, c1 = 64 * NB;
            if (by_keys) {
                stat_s[t][r] = make_float2(top, bad ? -sum : sum);   // a sum is not negative: its sign is a word from one stream to the other
                tc::bar_sync(3, 256);
                const float2 s0 = stat_s[0][r], s1 = stat_s[1][r];
                top = fmaxf(s0.x, s1.x);
                f[0] = s0.x == -INFINITY ? 0.f : ex2_approx((s0.x - top) * p.c);
                f[1] = s1.x == -INFINITY ? 0.f : ex2_approx((s1.x - top) * p.c);
                sum = f[0] * fabsf(s0.y) + f[1] * fabsf(s1.y);
                bad = signbit(s0.y) || signbit(s1.y);
                c0 = 32 * NB * t;
                c1 = c0 + 32 * NB;
            }
            for (int u = 0; u < 2; u++) {
                if (by_keys && j0 + u >= j1) continue;   // that stream had no tile
                if (by_keys || u == t) wait(b_o + 8 * u, no[u] & 1);
                no[u]++;
            }
            __syncwarp();
            tc::fence_after_sync();
            const bool cut = part.slot >= 0;
            const float inv = cut ? 1.f : sum != 0.f ? 1.f / sum : 0.f;   // nothing seen: 0
            const float g0 = f[0] * inv, g1 = f[1] * inv;
            const int64_t place = cut ? (int64_t)part.slot * p.rows + token * p.group + head : 0;
            uint16_t *out = reinterpret_cast<uint16_t *>(a.out.data) + (int64_t)(w.row0 + w.i0 + token) * a.out.token_stride + (int64_t)(w.kv_head * p.group + head) * a.out.head_stride;
            float *part_row = p.sums + place * a.c.width;
            if (some) {
                for (int c = c0; c < c1; c += 32) {
                    uint32_t o[32], o1[32];
                    __syncwarp();
                    if (by_keys || t == 0) tc::tmem_ld32(t_o + c, o);
                    if (by_keys || t == 1) tc::tmem_ld32(t_o + 128 + c, o1);
                    if (by_keys || t == 0) tc::tmem_ld_wait(o);
                    if (by_keys || t == 1) tc::tmem_ld_wait(o1);
                    // a stream that had no tile left what it found
#pragma unroll
                    for (int k = 0; k < 32; k++)
                        o[k] = __float_as_uint((f[0] != 0.f ? g0 * __uint_as_float(o[k]) : 0.f) + (f[1] != 0.f ? g1 * __uint_as_float(o1[k]) : 0.f));
                    if (!row) continue;
                    if (cut) {
#pragma unroll
                        for (int k = 0; k < 32; k += 4)
                            if (c + k < a.c.width) *reinterpret_cast<uint4 *>(part_row + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                    } else {
                        uint32_t y[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) y[k] = Half<T>::pack(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1]));
                        store_row32(out, y, c, a.c.width, p.wide);
                    }
                }
            }
            tc::fence_before_sync();
            tc::mbar_arrive(b_o_read);
            if (row) {
                if (cut && c0 == 0) p.stat[place] = make_float2(top * p.c, sum);
                if (bad) {
                    if (cut) poison_row<T>(p, part, pos, up, above, part_row, c0, min(c1, a.c.width));
                    else poison_row<T>(p, part, pos, up, above, out, c0, min(c1, a.c.width));
                }
            }
            x0 += 2 * (j1 - j0);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(b_part_free + 8 * slot_r);
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == PG_COPY) tc::tmem_dealloc(tmem, 512);
}

// Items that were cut: a warp a row, 4 columns a lane.  Parts lie in the CTAs from this one on, scaled here to their common maximum, in their order; one that has seen nothing has a sum of 0.
template <typename T>
__global__ void __launch_bounds__(256) paged_join(const __grid_constant__ PagedKernel p) {
    const PagedSplit s = p.split[blockIdx.x];
    const int row = 8 * blockIdx.y + (threadIdx.x >> 5), lane = threadIdx.x & 31, c = 4 * lane;
    if (row >= s.parts * p.rows || row >= s.w.tokens * p.group) return;
    auto place = [&](int i) { return (int64_t)(2 * ((int)blockIdx.x + i) + (i == 0)) * p.rows + row; };
    float high = -INFINITY, total = 0.f, o[4] = {};
    for (int i = lane; i < s.parts; i += 32) high = fmaxf(high, p.stat[place(i)].x);
#pragma unroll
    for (int x = 16; x; x >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
    if (c >= p.a.c.width) return;
    for (int i = 0; i < s.parts; i++) {
        const float2 t = p.stat[place(i)];
        if (t.y == 0.f) continue;
        const float f = ex2_approx(t.x - high);
        const float4 x = *reinterpret_cast<const float4 *>(p.sums + place(i) * p.a.c.width + c);
        total = fmaf(f, t.y, total);
        o[0] = fmaf(f, x.x, o[0]); o[1] = fmaf(f, x.y, o[1]); o[2] = fmaf(f, x.z, o[2]); o[3] = fmaf(f, x.w, o[3]);
    }
    const float inv = total != 0.f ? 1.f / total : 0.f;
    uint16_t *out = reinterpret_cast<uint16_t *>(p.a.out.data) + (int64_t)(s.w.row0 + s.w.i0 + row / p.group) * p.a.out.token_stride + (int64_t)(s.w.kv_head * p.group + row % p.group) * p.a.out.head_stride;
    *reinterpret_cast<uint2 *>(out + c) = make_uint2(Half<T>::pack(o[0] * inv, o[1] * inv), Half<T>::pack(o[2] * inv, o[3] * inv));
}

struct PagedGrid {
    int group, tokens, subs, ctas, rows;
    int64_t entries;
};
static PagedGrid paged_grid(const f3m_seqs &s, const f3m_cache &c, int heads) {
    PagedGrid g;
    g.group = heads / c.kv_heads;
    g.tokens = SEQ_TILE / g.group;
    g.subs = (std::min(s.longest, 2 * SEQ_TILE) + 2 * g.tokens - 1) / (2 * g.tokens);
    g.entries = (int64_t)s.pairs * g.subs;
    const int64_t most = ((int64_t)c.table_pages * c.page_tokens + s.longest) / SEQ_TILE + 1;   // tiles of keys of an item
    g.ctas = (int)std::min<int64_t>(NUM_SMS_HINT, std::min<int64_t>(g.entries * c.kv_heads, NUM_SMS_HINT) * most);
    g.rows = std::min(s.longest, 2 * g.tokens) * g.group;
    return g;
}
static size_t split_bytes(const PagedGrid &g) { return (g.ctas * sizeof(PagedSplit) + 15) / 16 * 16; }
size_t paged_workspace(const f3m_seqs &s, const f3m_cache &c, int heads) {
    if (heads / c.kv_heads > SEQ_TILE) return 0;
    const PagedGrid g = paged_grid(s, c, heads);
    return split_bytes(g) + 2 * (size_t)g.ctas * ((g.rows + 1) / 2 * 2) * (c.width + 2) * sizeof(float);
}

template <typename T>
static void paged_t(const PagedArgs &a, cudaStream_t s) {
    PagedKernel p;
    p.a = a;
    const PagedGrid g = paged_grid(a.s, a.c, a.heads);
    const int top = (int)std::min<int64_t>((int64_t)a.c.table_pages * a.c.page_tokens + a.s.longest, 0x7fffff00);   // no position is beyond
    p.a.window = std::min(a.window, std::max(top, 1));
    p.a.sinks = std::min(a.sinks, top);
    F3M_REQUIRE(g.entries <= 0x7fffffff - PG_THREADS, F3M_ERR_OVERFLOW, "%lld tiles of new tokens do not fit in 31 bits", (long long)g.entries);
    p.group = g.group; p.tokens = g.tokens; p.subs = g.subs; p.entries = (int)g.entries;
    p.rows = (g.rows + 1) / 2 * 2;
    p.page_shift = 31 - __builtin_clz(a.c.page_tokens);
    p.box = std::min(a.c.page_tokens, SEQ_TILE);
    p.wide = rows_wide(a.out);
    p.c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);   // a scale of zero: all weights are one
    p.err = seq_error_word();
    p.split = reinterpret_cast<PagedSplit *>(a.ws);
    p.sums = reinterpret_cast<float *>(reinterpret_cast<char *>(a.ws) + split_bytes(g));
    p.stat = reinterpret_cast<float2 *>(p.sums + 2 * (size_t)g.ctas * p.rows * a.c.width);
    p.mq = seq_tensor_map(Half<T>::type, a.q, a.s.tokens, a.heads, a.c.width, g.group, g.tokens);
    f3m_cache c = a.c;
    if (c.pages == 0) {   // no page is read: the maps need an address
        c.pages = 1;
        c.k = c.v = f3m_pages{a.q.data, c.width, c.width, c.width};
    }
    p.mk = page_tensor_map(Half<T>::type, c, c.k, p.box);
    p.mv = page_tensor_map(Half<T>::type, c, c.v, p.box);
    constexpr int blocks[2] = {2 + PG_SLOTS, 2 * (2 + 4)};
    const int bytes = blocks[a.c.width > 64] * PG_BLOCK + F3M_TREE_MAX * PG_WORDS * 4 + 1024;
    auto kernel = a.c.width <= 64 ? paged_tiles<T, 1> : paged_tiles<T, 2>;
    static SharedMemory allowed[2];
    allowed[a.c.width > 64].allow(kernel, bytes);
    kernel<<<g.ctas, PG_THREADS, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
    paged_join<T><<<dim3(g.ctas, (g.rows + 7) / 8), 256, 0, s>>>(p);
    F3M_LAUNCH_CHECK();
}

void paged_attention(int type, const PagedArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? paged_t<__nv_bfloat16>(a, s) : paged_t<__half>(a, s); }

// ---- accepted paths -----------------------------------------------------------------------------------------------------------
// A thread has 16 bytes of a row of keys or values and takes the places in order, KP_ROWS at a time: read, then written.  A place is read for one in front of it or
// for itself (kept[j] >= j), so that what is written has been read.
constexpr int KP_ROWS = 8, KP_THREADS = 128;
__global__ void __launch_bounds__(KP_THREADS) keep_paths(f3m_cache c, const int *kept, int64_t kept_stride, int most, const int *counts) {
    const int b = blockIdx.x, per = c.width / 8, x = blockIdx.y * KP_THREADS + threadIdx.x;
    if (x >= 2 * c.kv_heads * per) return;
    const f3m_pages &p = x < c.kv_heads * per ? c.k : c.v;
    const int h = x / per % c.kv_heads, col = 8 * (x % per), length = paged_length(c, b), count = min(max(counts[b], 0), most);
    uint16_t *data = reinterpret_cast<uint16_t *>(p.data) + col;
    for (int j0 = 0; j0 < count; j0 += KP_ROWS) {
        uint4 v[KP_ROWS];
        int64_t to[KP_ROWS];
#pragma unroll
        for (int r = 0; r < KP_ROWS; r++) {
            const int j = j0 + r;
            to[r] = -1;
            if (j >= count) continue;
            const int m = kept[b * kept_stride + j];
            if (m <= j) continue;   // its place already, or no place of a path
            const int page = paged_page(c, b, (int64_t)length + m), there = paged_page(c, b, (int64_t)length + j);
            if (page < 0 || there < 0) continue;
            to[r] = paged_at(c, p, there, (int64_t)length + j, h);
            v[r] = *reinterpret_cast<const uint4 *>(data + paged_at(c, p, page, (int64_t)length + m, h));
        }
#pragma unroll
        for (int r = 0; r < KP_ROWS; r++)
            if (to[r] >= 0) *reinterpret_cast<uint4 *>(data + to[r]) = v[r];
    }
}

void paged_keep(const f3m_cache &c, const int *kept, int64_t kept_stride, int most, const int *counts, cudaStream_t s) {
    keep_paths<<<dim3(c.sequences, (2 * c.kv_heads * (c.width / 8) + KP_THREADS - 1) / KP_THREADS), KP_THREADS, 0, s>>>(c, kept, kept_stride, most, counts);
    F3M_LAUNCH_CHECK();
}

}  // namespace f3m
