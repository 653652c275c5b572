// Attention over a window with sinks: forward, gradients, one new token against a cache.
#include <algorithm>
#include "packed.cuh"
#include "seq.cuh"

namespace f3m {

template <typename T>
__device__ __forceinline__ float dot_rows(const T *a, const T *b, int width, int lane) {
    float s = 0.f;
    for (int c = 2 * lane; c < width; c += 64) {
        const float2 x = Half<T>::unpack(*reinterpret_cast<const uint32_t *>(a + c)), y = Half<T>::unpack(*reinterpret_cast<const uint32_t *>(b + c));
        s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}
template <typename T>
__device__ __forceinline__ T *row_of(const f3m_rows &r, int64_t t, int h) { return reinterpret_cast<T *>(r.data) + t * r.token_stride + h * r.head_stride; }

// A warp per (query, head), the running maximum and sum of its softmax in registers.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(128) window_rows(WindowArgs a) {
    const int lane = threadIdx.x & 31, row = (blockIdx.x * 128 + threadIdx.x) >> 5, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[row / SEQ_TILE];
    const int i = e.z + row % SEQ_TILE;
    if (i >= e.y) return;
    const T *q = row_of<T>(a.q, e.x + i, h);
    float2 acc[2] = {};
    float top = -INFINITY, sum = 0.f, lse = 0.f, delta = 0.f;
    if (GRAD) {
        lse = a.lse[(int64_t)h * a.s.tokens + e.x + i];
        delta = dot_rows(row_of<T>(a.out, e.x + i, h), row_of<T>(a.dout, e.x + i, h), a.width, lane);
        if (lane == 0) a.delta[(int64_t)h * a.s.tokens + e.x + i] = delta;
    }
    const int lo = max(0, i - a.window + 1);
    for (int j = 0; j <= i; j++) {
        if (j < lo && j >= a.sinks) j = lo;
        const T *k = row_of<T>(a.k, e.x + j, hk), *v = row_of<T>(a.v, e.x + j, hk);
        const float s = a.scale * dot_rows(q, k, a.width, lane);
        float w, scale_acc = 1.f;
        if (GRAD) {
            w = expf(s - lse) * (dot_rows(row_of<T>(a.dout, e.x + i, h), v, a.width, lane) - delta) * a.scale;
        } else {
            const float t = fmaxf(top, s);
            scale_acc = expf(top - t);
            w = expf(s - t);
            top = t;
            sum = sum * scale_acc + w;
        }
        const T *src = GRAD ? k : v;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int c = 2 * lane + 64 * p;
            if (c < a.width) {
                const float2 x = Half<T>::unpack(*reinterpret_cast<const uint32_t *>(src + c));
                acc[p].x = acc[p].x * scale_acc + w * x.x;
                acc[p].y = acc[p].y * scale_acc + w * x.y;
            }
        }
    }
    const float inv = GRAD ? 1.f : 1.f / sum;
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const int c = 2 * lane + 64 * p;
        if (c < a.width) *reinterpret_cast<uint32_t *>(row_of<T>(GRAD ? a.dq : a.out, e.x + i, h) + c) = Half<T>::pack(acc[p].x * inv, acc[p].y * inv);
    }
    if (!GRAD && lane == 0) a.lse[(int64_t)h * a.s.tokens + e.x + i] = top + logf(sum);
}

// A warp per (key, key head): dk and dv are sums over the queries that see the key, of all heads that share it.
template <typename T>
__global__ void __launch_bounds__(128) window_cols(WindowArgs a) {
    const int lane = threadIdx.x & 31, row = (blockIdx.x * 128 + threadIdx.x) >> 5, hk = blockIdx.y, group = a.heads / a.kv_heads;
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[row / SEQ_TILE];
    const int j = e.z + row % SEQ_TILE;
    if (j >= e.y) return;
    const T *k = row_of<T>(a.k, e.x + j, hk), *v = row_of<T>(a.v, e.x + j, hk);
    float2 gk[2] = {}, gv[2] = {};
    const int hi = j < a.sinks ? e.y : (int)min((int64_t)e.y, (int64_t)j + a.window);
    for (int h = hk * group; h < (hk + 1) * group; h++)
        for (int i = j; i < hi; i++) {
            const T *q = row_of<T>(a.q, e.x + i, h), *g = row_of<T>(a.dout, e.x + i, h);
            const int64_t at = (int64_t)h * a.s.tokens + e.x + i;
            const float p = expf(a.scale * dot_rows(q, k, a.width, lane) - a.lse[at]);
            const float ds = p * (dot_rows(g, v, a.width, lane) - a.delta[at]) * a.scale;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int c = 2 * lane + 64 * r;
                if (c < a.width) {
                    const float2 x = Half<T>::unpack(*reinterpret_cast<const uint32_t *>(q + c)), y = Half<T>::unpack(*reinterpret_cast<const uint32_t *>(g + c));
                    gk[r].x = fmaf(ds, x.x, gk[r].x); gk[r].y = fmaf(ds, x.y, gk[r].y);
                    gv[r].x = fmaf(p, y.x, gv[r].x); gv[r].y = fmaf(p, y.y, gv[r].y);
                }
            }
        }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int c = 2 * lane + 64 * r;
        if (c < a.width) {
            *reinterpret_cast<uint32_t *>(row_of<T>(a.dk, e.x + j, hk) + c) = Half<T>::pack(gk[r].x, gk[r].y);
            *reinterpret_cast<uint32_t *>(row_of<T>(a.dv, e.x + j, hk) + c) = Half<T>::pack(gv[r].x, gv[r].y);
        }
    }
}

// ---- forward --------------------------------------------------------------------------------------------------------------
// A CTA, one per SM, walks over items; an item is two tiles of 128 query rows that read the same keys: two heads of a group, or, where a group has
// an odd number of heads, two neighbouring tiles of one head.  Tile by tile of 128 keys, S = Q K^T goes to tensor memory; a thread has one
// row of S, takes the weights 2^(c s - c top) and writes them, rounded to 16 bits, over S, from where they go into O += P V.  While one
// query tile's weights are taken, the other's products run.
//
// `top` follows the row's maximum lazily: weights are at most 2^8, and O in tensor memory is only scaled when the maximum has risen by more than
// that since the last time.  The row sum is taken in FP32 before the weights are rounded.
//
// What bounds it: 128 x 128 exponentials a tile at 16 a clock and SM take 1024 clocks, its two products at width 128 as many.
constexpr int WF_COPY = 8, WF_PRODUCTS = 9, WF_THREADS = 320, WF_BLOCK = SEQ_TILE * 128;
constexpr int WF_BLOCKS = 14;      // blocks of 64 columns: two query tiles, a ring of key and value tiles, two to stage outputs

struct WindowKernel {
    WindowArgs a;
    CUtensorMap mq, mk, mv, mo;
    int items;
    bool by_heads;      // an item's tiles are two heads of a group, else two neighbouring tiles of a head
    float c;            // |scale| log2(e)
    int *err;
};
struct WindowItem {
    int row0, len, start, head[2], kv_head, tiles_q;   // tile t: tokens from start + (by_heads ? 0 : 128 t) on
    int sinks, first, keys;                            // tiles of keys: the first `sinks` of the sequence, then those from tile `first` on; `keys` in all
    __device__ __forceinline__ int key(int j) const { return SEQ_TILE * (j < sinks ? j : first + j - sinks); }
};
__device__ __forceinline__ WindowItem window_item(const WindowKernel &p, int i) {
    const WindowArgs &a = p.a;
    const int group = a.heads / a.kv_heads;
    WindowItem w;
    int4 e;
    int last;
    if (p.by_heads) {
        const int n = a.heads / 2, pair = i % n;
        e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_past(a.s, i / n)];
        w.head[0] = 2 * pair; w.head[1] = 2 * pair + 1;
        w.tiles_q = 2;
        last = min(e.y, e.z + SEQ_TILE) - 1;
    } else {
        const int h = i % a.heads;
        e = reinterpret_cast<const int4 *>(a.s.table)[seq_pair_by_past(a.s, i / a.heads)];
        w.head[0] = w.head[1] = h;
        w.tiles_q = e.y - e.z > SEQ_TILE ? 2 : 1;
        last = min(e.y, e.z + 2 * SEQ_TILE) - 1;
    }
    w.kv_head = w.head[0] / group;
    w.row0 = e.x; w.len = e.y; w.start = e.z;
    w.first = max(0, e.z - a.window + 1) / SEQ_TILE;
    w.sinks = (int)min(((int64_t)a.sinks + SEQ_TILE - 1) / SEQ_TILE, (int64_t)w.first);
    w.keys = w.sinks + last / SEQ_TILE - w.first + 1;
    return w;
}

template <typename T>
__global__ void __launch_bounds__(WF_THREADS, 1) window_tiles(const __grid_constant__ WindowKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 8 + 2 + 8];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    const WindowArgs &a = p.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nb = (a.width + 63) / 64;
    const int slots = min(8, (WF_BLOCKS - 2 * nb - 2) / nb);   // 4 at two blocks, 8 at one
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u;
    auto q_tile = [&](int t) { return smem + t * nb * WF_BLOCK; };
    auto slot_tile = [&](int s) { return smem + (2 + s) * nb * WF_BLOCK; };
    const uint32_t stage = smem + (2 + slots) * nb * WF_BLOCK;

    if (warp == WF_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    if (tid == 0) {
        for (int i = 0; i < 18; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);        // slot landed, free; queries landed, free
        for (int t = 0; t < 2; t++) {
            tc::mbar_init(tc::smem_u32(&bars[18 + t]), 1);      // S ready
            tc::mbar_init(tc::smem_u32(&bars[20 + t]), 128);    // weights written
            tc::mbar_init(tc::smem_u32(&bars[22 + t]), 1);      // O ready
            tc::mbar_init(tc::smem_u32(&bars[24 + t]), 128);    // O read
        }
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s;
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[8]), b_q = tc::smem_u32(&bars[16]), b_q_free = tc::smem_u32(&bars[17]),
                   b_s = tc::smem_u32(&bars[18]), b_p = tc::smem_u32(&bars[20]), b_o = tc::smem_u32(&bars[22]), b_o_read = tc::smem_u32(&bars[24]);

    if (warp == WF_COPY) {
        if (lane == 0) {
            int x = 0, items = 0;   // key and value tiles so far, items so far
            for (int it = blockIdx.x; it < p.items && !gave_up_s; it += gridDim.x, items++) {
                const WindowItem w = window_item(p, it);
                if (items) wait(b_q_free, (items - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_q, w.tiles_q * nb * WF_BLOCK);
                for (int t = 0; t < w.tiles_q; t++)
                    for (int k = 0; k < nb; k++)
                        tc::tma_rows(q_tile(t) + k * WF_BLOCK, &p.mq, 64 * k, w.head[t], w.row0 + w.start + (p.by_heads ? 0 : t * SEQ_TILE), b_q);
                for (int j = 0; j < 2 * w.keys && !gave_up_s; j++, x++) {
                    const int s = x % slots;
                    if (x >= slots) wait(b_free + 8 * s, (x / slots - 1) & 1);
                    if (gave_up_s) break;
                    tc::mbar_expect_tx(b_full + 8 * s, nb * WF_BLOCK);
                    for (int k = 0; k < nb; k++) tc::tma_rows(slot_tile(s) + k * WF_BLOCK, j & 1 ? &p.mv : &p.mk, 64 * k, w.kv_head, w.row0 + w.key(j >> 1), b_full + 8 * s);
                }
            }
            for (int s = 0; s < slots; s++)   // the last copies
                if (x > s) wait.drain(b_full + 8 * s, ((x - 1 - s) / slots) & 1);
            if (items) wait.drain(b_q, (items - 1) & 1);
        }
    } else if (warp == WF_PRODUCTS) {
        if (lane == 0) {
            constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
            // a negative scale turns S's sign: bit 13 negates A
            const uint32_t i_s = tc::idesc_f16(bf, 128, 128, false, false) | (a.scale < 0.f ? 1u << 13 : 0u), i_o = tc::idesc_f16(bf, 128, 64 * nb, false, true);
            int x = 0, items = 0, np[2] = {0, 0}, no[2] = {0, 0};
            auto scores = [&](int t, int s) {
                for (int k = 0; k < 4 * nb; k++)
                    tc::mma_f16(tmem + 128 * t, tc::desc_k(q_tile(t) + (k >> 2) * WF_BLOCK + (k & 3) * 32), tc::desc_k(slot_tile(s) + (k >> 2) * WF_BLOCK + (k & 3) * 32), i_s, k > 0);
                tc::mma_commit(b_s + 8 * t);
            };
            for (int it = blockIdx.x; it < p.items; it += gridDim.x, items++) {
                const WindowItem w = window_item(p, it);
                wait(b_q, items & 1);
                int sk = x % slots;
                wait(b_full + 8 * sk, (x / slots) & 1);
                tc::fence_after_sync();
                for (int t = 0; t < w.tiles_q; t++) scores(t, sk);
                tc::mma_commit(b_free + 8 * sk);
                if (w.keys == 1) tc::mma_commit(b_q_free);
                for (int j = 0; j < w.keys; j++) {
                    const int xv = x + 2 * j + 1, sv = xv % slots;
                    const bool more = j + 1 < w.keys;
                    sk = (xv + 1) % slots;
                    for (int t = 0; t < w.tiles_q; t++) {
                        if (t == 0) wait(b_full + 8 * sv, (xv / slots) & 1);
                        if (j == 0 && no[t]) wait(b_o_read + 8 * t, (no[t] - 1) & 1);
                        wait(b_p + 8 * t, np[t] & 1);
                        np[t]++;
                        tc::fence_after_sync();
                        for (int k = 0; k < 8; k++) tc::mma_f16_ta(tmem + 256 + 128 * t, tmem + 128 * t + 8 * k, tc::desc_mn(slot_tile(sv) + k * 2048, WF_BLOCK), i_o, j > 0 || k > 0);
                        if (more) {
                            if (t == 0) {
                                wait(b_full + 8 * sk, ((xv + 1) / slots) & 1);
                                tc::fence_after_sync();
                            }
                            scores(t, sk);
                        } else {
                            tc::mma_commit(b_o + 8 * t);
                            no[t]++;
                        }
                    }
                    tc::mma_commit(b_free + 8 * sv);
                    if (more) tc::mma_commit(b_free + 8 * sk);
                    if (j + 2 == w.keys) tc::mma_commit(b_q_free);
                }
                x += 2 * w.keys;
            }
        }
    } else {
        // ---- weights: thread r of a query tile has its row r ----
        const int t = warp >> 2, r = tid & 127, wq = warp & 3;
        const uint32_t lanes = (uint32_t)(32 * wq) << 16, t_s = tmem + 128 * t + lanes, t_o = tmem + 256 + 128 * t + lanes;
        int ns = 0, no = 0, x = 0;
        for (int it = blockIdx.x; it < p.items; it += gridDim.x) {
            const WindowItem w = window_item(p, it);
            if (t < w.tiles_q) {   // whole warps
                const int start = w.start + (p.by_heads ? 0 : t * SEQ_TILE), i = start + r, i0 = start + 32 * wq;
                float top = -INFINITY, sum = 0.f;
                for (int j = 0; j < w.keys; j++) {
                    const int key = w.key(j);
                    wait(b_s + 8 * t, ns & 1);
                    ns++;
                    __syncwarp();
                    tc::fence_after_sync();
                    // a row sees the keys j <= i of the window, i - j < window, and the sinks; most tiles are seen whole.  S is read twice,
                    // for the maximum and for the weights: 128 scores and their weights do not fit in the registers beside the rest.
                    const bool whole = key + SEQ_TILE - 1 <= i0 && (i0 + 31 - key < a.window || key + SEQ_TILE <= a.sinks);
                    const int up = i - key, low = i - key - a.window, sink = a.sinks - key;   // seen: c <= up and (c > low or c < sink)
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int q = 0; q < 4; q += 2) {
                        uint32_t s0[32], s1[32];
                        tc::tmem_ld32(t_s + 32 * q, s0);
                        tc::tmem_ld32(t_s + 32 * q + 32, s1);
                        tc::tmem_ld_wait(s0);
                        tc::tmem_ld_wait(s1);
                        if (whole) {
#pragma unroll
                            for (int c = 0; c < 32; c++) {
                                mx[2 * (c & 1)] = fmaxf(mx[2 * (c & 1)], __uint_as_float(s0[c]));
                                mx[2 * (c & 1) + 1] = fmaxf(mx[2 * (c & 1) + 1], __uint_as_float(s1[c]));
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < 32; c++) {
                                const int c0 = 32 * q + c, c1 = c0 + 32;
                                mx[2 * (c & 1)] = fmaxf(mx[2 * (c & 1)], c0 <= up && (c0 > low || c0 < sink) ? __uint_as_float(s0[c]) : -INFINITY);
                                mx[2 * (c & 1) + 1] = fmaxf(mx[2 * (c & 1) + 1], c1 <= up && (c1 > low || c1 < sink) ? __uint_as_float(s1[c]) : -INFINITY);
                            }
                        }
                    }
                    const float high = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                    const bool rise = (high - top) * p.c > 8.f;   // also from -inf; not from -inf to -inf
                    if (__any_sync(0xffffffffu, rise)) {
                        const float f = rise ? exp2_approx((top - high) * p.c) : 1.f;
                        if (rise) { top = high; sum *= f; }
                        if (j > 0)
                            for (int q = 0; q < 2 * nb; q++) {
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
                    f32x2 part[2] = {pack2(sum, 0.f), pack2(0.f, 0.f)};
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        uint32_t x[32], w16[16];
                        tc::tmem_ld32(t_s + 32 * q, x);
                        tc::tmem_ld_wait(x);
                        if (!whole)
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (!(32 * q + c <= up && (32 * q + c > low || 32 * q + c < sink))) x[c] = 0xff800000u;
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float lo, hi;
                            unpack2(fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), cc, ss), lo, hi);
                            lo = ex2_approx(lo);
                            hi = ex2_approx(hi);
                            part[(c >> 1) & 1] = add2(part[(c >> 1) & 1], pack2(lo, hi));
                            w16[c >> 1] = Half<T>::pack(lo, hi);
                        }
                        tc::tmem_st16(t_s + 16 * q, w16);   // over scores that have been read
                    }
                    float u, v;
                    unpack2(add2(part[0], part[1]), u, v);
                    sum = u + v;
                    if (t == 0 && key + SEQ_TILE > w.len) {   // the sequence ends inside the tile
                        const int xv = x + 2 * j + 1, sv = xv % slots;
                        wait(b_full + 8 * sv, (xv / slots) & 1);
                        if (key + r >= w.len) clear_row(slot_tile(sv), r, 0, 8 * nb);
                        tc::fence_async_smem();
                        __syncwarp();
                    }
                    tc::tmem_st_wait();
                    tc::fence_before_sync();
                    tc::mbar_arrive(b_p + 8 * t);
                }
                wait(b_o + 8 * t, no & 1);
                no++;
                __syncwarp();
                tc::fence_after_sync();
                const int m = min(SEQ_TILE, w.len - start);
                const float inv = 1.f / sum;
                for (int q = 0; q < 2 * nb; q++) {
                    uint32_t o[32];
                    __syncwarp();
                    tc::tmem_ld32(t_o + 32 * q, o);
                    tc::tmem_ld_wait(o);
                    if (q + 1 == 2 * nb) {
                        tc::fence_before_sync();
                        tc::mbar_arrive(b_o_read + 8 * t);
                    }
#pragma unroll
                    for (int c = 0; c < 32; c += 8) {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) y[k] = Half<T>::pack(inv * __uint_as_float(o[c + 2 * k]), inv * __uint_as_float(o[c + 2 * k + 1]));
                        sts16(stage + t * WF_BLOCK + tc::swz(r, 4 * (q & 1) + c / 8), y);
                    }
                    if (q & 1) {
                        store_rows<128>(p.mo, a.out, stage + t * WF_BLOCK, w.head[t], w.row0 + start, m, 32 * (q - 1), 1, a.width, r, 1 + t);
                        tc::bar_sync(1 + t, 128);   // the block may be written again
                    }
                }
                if (r < m) a.lse[(int64_t)w.head[t] * a.s.tokens + w.row0 + i] = (top * p.c + log2f(sum)) * 0.69314718055994531f;
            }
            x += 2 * w.keys;
        }
        if (r == 0) tc::tma_store_wait_all();
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == WF_COPY) tc::tmem_dealloc(tmem, 512);
}

template <typename T>
static void forward_t(const WindowArgs &a, cudaStream_t s) {
    WindowKernel p;
    p.a = a;
    p.a.window = std::min(a.window, a.s.longest);   // places and their differences stay within 31 bits
    p.a.sinks = std::min(a.sinks, a.s.longest);
    p.mq = seq_tensor_map(Half<T>::type, a.q, a.s.tokens, a.heads, a.width);
    p.mk = seq_tensor_map(Half<T>::type, a.k, a.s.tokens, a.kv_heads, a.width);
    p.mv = seq_tensor_map(Half<T>::type, a.v, a.s.tokens, a.kv_heads, a.width);
    p.mo = seq_tensor_map(Half<T>::type, a.out, a.s.tokens, a.heads, a.width);
    p.by_heads = a.heads / a.kv_heads % 2 == 0;
    const int64_t items = p.by_heads ? (int64_t)a.s.tiles * (a.heads / 2) : (int64_t)a.s.pairs * a.heads;
    F3M_REQUIRE(items <= 0x7fffffff - NUM_SMS_HINT, F3M_ERR_OVERFLOW, "%d tiles of %d heads do not fit in 31 bits", a.s.tiles, a.heads);
    p.items = (int)items;
    p.c = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1e-30f);   // a scale of zero: all weights are one
    p.err = seq_error_word();
    constexpr int bytes = WF_BLOCKS * WF_BLOCK + 1024;
    F3M_CUDA(cudaFuncSetAttribute(window_tiles<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    window_tiles<T><<<std::min(p.items, NUM_SMS_HINT), WF_THREADS, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
}
template <typename T>
static void backward_t(const WindowArgs &a, cudaStream_t s) {
    window_rows<T, true><<<dim3(a.s.tiles * 32, a.heads), 128, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
    window_cols<T><<<dim3(a.s.tiles * 32, a.kv_heads), 128, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}
void window_forward(int type, const WindowArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? forward_t<__nv_bfloat16>(a, s) : forward_t<__half>(a, s); }
void window_backward(int type, const WindowArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? backward_t<__nv_bfloat16>(a, s) : backward_t<__half>(a, s); }

// A warp per (sequence, head) reads the keys that are seen one by one.
template <typename T>
__global__ void __launch_bounds__(32) step_rows(StepArgs a) {
    const int lane = threadIdx.x, b = blockIdx.x, h = blockIdx.y, hk = h / (a.heads / a.kv_heads);
    const int len = min(max(a.lengths[b], 0), (int)a.capacity), lo = max(0, len - a.window);
    const T *q = row_of<T>(a.q, b, h);
    float2 acc[2] = {};
    float top = -INFINITY, sum = 0.f;
    for (int j = 0; j < len; j++) {
        if (j < lo && j >= a.sinks) j = lo;
        const T *k = row_of<T>(a.k, j, hk) + b * a.k_seq, *v = row_of<T>(a.v, j, hk) + b * a.v_seq;
        const float s = a.scale * dot_rows(q, k, a.width, lane), t = fmaxf(top, s), old = expf(top - t), w = expf(s - t);
        top = t;
        sum = sum * old + w;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            const int c = 2 * lane + 64 * p;
            if (c < a.width) {
                const float2 x = Half<T>::unpack(*reinterpret_cast<const uint32_t *>(v + c));
                acc[p].x = acc[p].x * old + w * x.x;
                acc[p].y = acc[p].y * old + w * x.y;
            }
        }
    }
    const float inv = len ? 1.f / sum : 0.f;
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const int c = 2 * lane + 64 * p;
        if (c < a.width) *reinterpret_cast<uint32_t *>(row_of<T>(a.out, b, h) + c) = Half<T>::pack(acc[p].x * inv, acc[p].y * inv);
    }
}
int window_step_parts(int, int, int, int64_t, int, int) { return 1; }
size_t window_step_part_floats(int, int, int, int) { return 0; }
void window_step(int type, const StepArgs &a, cudaStream_t s) {
    if (type == F3M_TYPE_BF16) step_rows<__nv_bfloat16><<<dim3(a.n, a.heads), 32, 0, s>>>(a);
    else step_rows<__half><<<dim3(a.n, a.heads), 32, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}

}  // namespace f3m
