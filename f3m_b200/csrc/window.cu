// Attention over a window with sinks: forward, gradients, one new token against a cache.
#include <algorithm>
#include "seq.cuh"

namespace f3m {

template <typename T>
__device__ __forceinline__ T *row_of(const f3m_rows &r, int64_t t, int h) { return reinterpret_cast<T *>(r.data) + t * r.token_stride + h * r.head_stride; }

// ---- forward --------------------------------------------------------------------------------------------------------------
// A CTA, one per SM, walks over items; an item is two tiles of 128 query rows that read the same keys: two heads of a group, or, where a group has
// an odd number of heads, two neighbouring tiles of one head.  Tile by tile of 128 keys, S = Q K^T goes to tensor memory; a thread has one
// row of S, takes the weights 2^(c s - c top) and writes them, rounded to 16 bits, over S, from where they go into O += P V.  While one
// query tile's weights are taken, the other's products run.
//
// `top` follows the row's maximum lazily: weights are at most 2^8, and O in tensor memory is only scaled when the maximum has risen by more than
// that since the last time.  The row sum is taken in FP32 before the weights are rounded.
//
// What bounds it: 128 x 128 exponentials a tile at 16 a clock and SM take 1024 clocks, its two products at width 128 as many.  A quarter of the
// exponentials goes to the FMA pipe (an eighth: 522 us, half: 544), and the values' product begins at the first half of the weights; what is
// left is a tile's chain -- scores 1250 clocks, maximum 370, exponentials 1300 -- of which two run side by side.  16384 tokens, 16 heads on 4, width 128,
// window 4096: 505-535 us from box to box, 0.90-0.95 PFLOP/s, 56 % of measured; tensor pipe 49 % busy, issue slots 44 %.
//
// Here and in the other kernels one thread issues a block's products, and a product that overwrites scores follows the one that reads its weights
// from their columns with no wait between.  PTX promises the order of products of one accumulator and shape; that others too run one behind the other is
// relied on, and what repeated calls' equal bits are tested for.
constexpr int WF_COPY = 8, WF_PRODUCTS = 9, WF_THREADS = 320, WF_BLOCK = SEQ_TILE * 128;
constexpr float NO_SUM = 0x1p60f;  // no sum of 2^31 weights comes near: some exponent was not a number (exp2_poly)
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
    // Whether some query of the tile from `from` on sees some key of the tile from k on.  Of two neighbouring tiles one may not: its weights are zeros, and stay out
    // of its product, as a zero times what is not finite is no zero.
    __device__ __forceinline__ bool sees(const WindowArgs &a, int from, int k) const {
        return k < from + SEQ_TILE && (k < a.sinks || from - k - (SEQ_TILE - 1) < a.window);
    }
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

template <typename T, int NB>
__global__ void __launch_bounds__(WF_THREADS, 1) window_tiles(const __grid_constant__ WindowKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 8 + 2 + 11];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    const WindowArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int slots = NB == 2 ? 4 : 8;
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u;
    auto q_tile = [&](int t) { return smem + t * NB * WF_BLOCK; };
    auto slot_tile = [&](int s) { return smem + (2 + s) * NB * WF_BLOCK; };
    const uint32_t stage = smem + (2 + slots) * NB * WF_BLOCK;

    if (warp == WF_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    if (tid == 0) {
        for (int i = 0; i < 18; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);        // slot landed, free; queries landed, free
        for (int t = 0; t < 2; t++) {
            tc::mbar_init(tc::smem_u32(&bars[18 + t]), 1);      // S ready
            tc::mbar_init(tc::smem_u32(&bars[20 + t]), 128);    // weights of the first 64 keys written
            tc::mbar_init(tc::smem_u32(&bars[22 + t]), 1);      // O ready
            tc::mbar_init(tc::smem_u32(&bars[24 + t]), 128);    // O read
            tc::mbar_init(tc::smem_u32(&bars[26 + t]), 128);    // weights of the other 64 written
        }
        tc::mbar_init(tc::smem_u32(&bars[28]), 1);              // no products in flight
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s;
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[8]), b_q = tc::smem_u32(&bars[16]), b_q_free = tc::smem_u32(&bars[17]),
                   b_s = tc::smem_u32(&bars[18]), b_p = tc::smem_u32(&bars[20]), b_o = tc::smem_u32(&bars[22]), b_o_read = tc::smem_u32(&bars[24]), b_p2 = tc::smem_u32(&bars[26]);

    if (warp == WF_COPY) {
        if (lane == 0) {
            int x = 0, items = 0;   // key and value tiles so far, items so far
            for (int it = blockIdx.x; it < p.items && !gave_up_s; it += gridDim.x, items++) {
                const WindowItem w = window_item(p, it);
                if (items) wait(b_q_free, (items - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_q, w.tiles_q * NB * WF_BLOCK);
                for (int t = 0; t < w.tiles_q; t++)
                    for (int k = 0; k < NB; k++)
                        tc::tma_rows(q_tile(t) + k * WF_BLOCK, &p.mq, 64 * k, w.head[t], w.row0 + w.start + (p.by_heads ? 0 : t * SEQ_TILE), b_q);
                for (int j = 0; j < 2 * w.keys && !gave_up_s; j++, x++) {
                    const int s = x % slots;
                    if (x >= slots) wait(b_free + 8 * s, (x / slots - 1) & 1);
                    if (gave_up_s) break;
                    tc::mbar_expect_tx(b_full + 8 * s, NB * WF_BLOCK);
                    for (int k = 0; k < NB; k++) tc::tma_rows(slot_tile(s) + k * WF_BLOCK, j & 1 ? &p.mv : &p.mk, 64 * k, w.kv_head, w.row0 + w.key(j >> 1), b_full + 8 * s);
                }
            }
            for (int s = 0; s < slots; s++)   // the last copies
                if (x > s) wait.drain(b_full + 8 * s, ((x - 1 - s) / slots) & 1);
            if (items) wait.drain(b_q, (items - 1) & 1);
        }
    } else if (warp == WF_PRODUCTS) {
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        // a negative scale turns S's sign: bit 13 negates A
        const uint32_t i_s = tc::idesc_f16(bf, 128, 128, false, false) | (a.scale < 0.f ? 1u << 13 : 0u), i_o = tc::idesc_f16(bf, 128, 64 * NB, false, true);
        int x = 0, items = 0, np[2] = {0, 0}, no[2] = {0, 0};
        for (int it = blockIdx.x; it < p.items; it += gridDim.x, items++) {
            const WindowItem w = window_item(p, it);
            wait(b_q, items & 1);
            int sk = x % slots;
            wait(b_full + 8 * sk, (x / slots) & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                for (int t = 0; t < w.tiles_q; t++) {
                    tc::product_rows<NB>(tmem + 128 * t, q_tile(t), slot_tile(sk), i_s);
                    tc::mma_commit(b_s + 8 * t);
                }
                tc::mma_commit(b_free + 8 * sk);
                if (w.keys == 1) tc::mma_commit(b_q_free);
            }
            bool begun[2] = {false, false};
            for (int j = 0; j < w.keys; j++) {
                const int xv = x + 2 * j + 1, sv = xv % slots;
                const bool more = j + 1 < w.keys;
                sk = (xv + 1) % slots;
                wait(b_full + 8 * sv, (xv / slots) & 1);
                if (more) wait(b_full + 8 * sk, ((xv + 1) / slots) & 1);
                for (int t = 0; t < w.tiles_q; t++) {
                    const bool seen = p.by_heads || w.sees(a, w.start + t * SEQ_TILE, w.key(j));
                    if (j == 0 && no[t]) wait(b_o_read + 8 * t, (no[t] - 1) & 1);
                    wait(b_p + 8 * t, np[t] & 1);
                    tc::fence_after_sync();
                    if (seen && tc::elect()) {
                        tc::product_tmem64(tmem + 256 + 128 * t, tmem + 128 * t, slot_tile(sv), i_o, begun[t]);
                    }
                    wait(b_p2 + 8 * t, np[t] & 1);
                    np[t]++;
                    no[t] += !more;
                    tc::fence_after_sync();
                    if (tc::elect()) {
                        if (seen) tc::product_tmem64(tmem + 256 + 128 * t, tmem + 128 * t + 32, slot_tile(sv) + 64 * 128, i_o, 1);
                        if (more) {
                            tc::product_rows<NB>(tmem + 128 * t, q_tile(t), slot_tile(sk), i_s);
                            tc::mma_commit(b_s + 8 * t);
                        } else {
                            tc::mma_commit(b_o + 8 * t);
                        }
                    }
                    begun[t] |= seen;
                }
                if (tc::elect()) {
                    tc::mma_commit(b_free + 8 * sv);
                    if (more) tc::mma_commit(b_free + 8 * sk);
                    if (j + 2 == w.keys) tc::mma_commit(b_q_free);
                }
            }
            x += 2 * w.keys;
        }
        wait.drain_products(tc::smem_u32(&bars[28]));
    } else {
        // ---- weights: thread r of a query tile has its row r ----
        const int t = warp >> 2, r = tid & 127, wq = warp & 3;
        const uint32_t lanes = (uint32_t)(32 * wq) << 16, t_s = tmem + 128 * t + lanes, t_o = tmem + 256 + 128 * t + lanes;
        int ns = 0, no = 0, x0 = 0;   // x0: key and value tiles of the items before
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
                    // for the maximum and for the weights, 32 columns at a time (146 registers); 128 scores held between the two were not tried.
                    const bool whole = key + SEQ_TILE - 1 <= i0 && (i0 + 31 - key < a.window || key + SEQ_TILE <= a.sinks);
                    const int up = i - key, low = i - key - a.window, sink = a.sinks - key;   // seen: c <= up and (c > low or c < sink)
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
                            for (int c = 0; c < 32; c++)
                                mx[c & 3] = fmaxf(mx[c & 3], 32 * q + c <= up && (32 * q + c > low || 32 * q + c < sink) ? __uint_as_float(x[q & 1][c]) : -INFINITY);
                        }
                    }
                    tc::tmem_ld32(t_s, x[0]);   // again
                    const float high = fmaxf(top, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
                    const bool rise = (high - top) * p.c > 8.f;   // also from -inf; not from -inf to -inf
                    if (__any_sync(0xffffffffu, rise)) {
                        const float f = rise ? ex2_approx((top - high) * p.c) : 1.f;
                        if (rise) { top = high; sum = sum < NO_SUM ? sum * f : NAN; }
                        if (j > 0)
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
                    f32x2 part[2] = {pack2(sum, 0.f), pack2(0.f, 0.f)};
                    if (t == 0 && key + SEQ_TILE > w.len) {   // the sequence ends inside the tile
                        const int xv = x0 + 2 * j + 1, sv = xv % slots;
                        wait(b_full + 8 * sv, (xv / slots) & 1);
                        if (key + r >= w.len) clear_row(slot_tile(sv), r, 0, 8 * NB);
                        tc::fence_async_smem();
                        __syncwarp();
                    }
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
                                part[(c >> 1) & 1] = add2(part[(c >> 1) & 1], pack2(lo, hi));
                                w16[c >> 1] = Half<T>::pack(lo, hi);
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < 32; c += 2) {
                                float lo, hi;
                                unpack2(fma2(pack2(__uint_as_float(y[c]), __uint_as_float(y[c + 1])), cc, ss), lo, hi);
                                const int c0 = 32 * q + c, c1 = c0 + 1;
                                lo = c0 <= up && (c0 > low || c0 < sink) ? ex2_approx(lo) : 0.f;
                                hi = c1 <= up && (c1 > low || c1 < sink) ? ex2_approx(hi) : 0.f;
                                part[(c >> 1) & 1] = add2(part[(c >> 1) & 1], pack2(lo, hi));
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
                    unpack2(add2(part[0], part[1]), u, v);
                    sum = u + v;
                }
                wait(b_o + 8 * t, no & 1);
                no++;
                __syncwarp();
                tc::fence_after_sync();
                const int m = min(SEQ_TILE, w.len - start);
                if (!isfinite(top) || !(sum < NO_SUM)) sum = NAN;
                const float inv = 1.f / sum;
                for (int q = 0; q < 2 * NB; q++) {
                    uint32_t o[32];
                    __syncwarp();
                    tc::tmem_ld32(t_o + 32 * q, o);
                    tc::tmem_ld_wait(o);
                    if (q + 1 == 2 * NB) {
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
            x0 += 2 * w.keys;
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
    auto kernel = a.width <= 64 ? window_tiles<T, 1> : window_tiles<T, 2>;
    static SharedMemory allowed[2];
    allowed[a.width > 64].allow(kernel, bytes);
    kernel<<<std::min(p.items, NUM_SMS_HINT), WF_THREADS, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
}
// ---- gradients ------------------------------------------------------------------------------------------------------------
// P = 2^(c s - lse), dS = P (dP - delta) with dP = dout V^T: dV = P^T dout, dK = scale dS^T Q, dQ = scale dS K.  dK and dV are sums over queries, dQ
// over keys: two kernels, one that holds a tile of keys and walks over the queries that see it, of all heads that share it, and one that
// holds a tile of queries.  S and dP are computed in both, seven products where five would do, but nothing is added across CTAs: sums have one order.
// P and dS are rounded to 16 bits where they become operands, and go through tensor memory over the scores they come from.
// What bounds it: a tile pair's weights and dS, some 3300 clocks for 256 threads; its products take 2048 (four) and 1536 (three).  2 x 4096 tokens, 8 heads,
// width 128, window 2048, forward and gradients: 305-320 us, 0.55 PFLOP/s by the formula's products, 0.72 by those computed; tensor pipe 53 % busy.

// fp16 ends at 2^-24, and dS is far smaller than dout: it would lose its bits where dout still has them (dout of 1e-4: dq and dk were 3 % off).  There P is
// taken times 2^15 and dS times 2^k, k from the largest |dout_i| and |v_j| of the sequence and the heads that share v: |dP - delta| <= 2 |dout_i| max |v_j|, as out_i
// is a mean of v_j, and dS stays below 2^15.  The powers of two leave in FP32, where gradients are stored.  bf16 has FP32's range and takes neither.
template <typename T> constexpr int WG_P_EXP = Half<T>::type == F3M_TYPE_F16 ? 15 : 0;
struct GradRange {
    float ds;           // what dP and delta are multiplied by beside P 2^15
    float out_s, out_v; // what dQ, dK and dV are multiplied by at the end
};
// range: squares of the largest finite |dout_i| and |v_j|
template <typename T>
__device__ __forceinline__ GradRange grad_range(const float *range, int kv_heads, int seq, int hk, float scale) {
    if constexpr (WG_P_EXP<T> == 0) return {1.f, scale, 1.f};
    const float2 r = reinterpret_cast<const float2 *>(range)[(int64_t)seq * kv_heads + hk];
    const float most = 2.f * sqrtf(r.x) * sqrtf(r.y);
    const int k = most > 0.f ? 14 - ((int)(__float_as_uint(most) >> 23) - 127) : 0;   // 2^(14 - k) <= most < 2^(15 - k); -26 <= k <= 62
    auto power = [](int e) { return __uint_as_float((uint32_t)(e + 127) << 23); };
    return {power(k - WG_P_EXP<T>), scale * power(-k), power(-WG_P_EXP<T>)};
}
// lse2 = lse log2(e), less the power of two of P, and delta = dout.out, rows (heads, tokens); in fp16 the range too.  A CTA has 64 of the
// rows of a tile of tokens and the query heads that share a key head, 16 threads a row.
template <typename T>
__global__ void __launch_bounds__(256) window_rows_sum(const __grid_constant__ WindowArgs a, float *lse2, float *delta, uint32_t *range) {
    const int group = a.heads / a.kv_heads, hk = blockIdx.x % a.kv_heads, c = 8 * (threadIdx.x & 15);
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, blockIdx.x / a.kv_heads)];
    const int64_t t0 = (int64_t)e.x + e.z;
    const int m = min(SEQ_TILE, e.y - e.z), rows = m * group;
    auto read = [&](const f3m_rows &r, int64_t t, int h, bool in) { return in ? *reinterpret_cast<const uint4 *>(row_of<T>(r, t, h) + c) : make_uint4(0u, 0u, 0u, 0u); };
    auto dot = [](const uint4 &x, const uint4 &y) {
        const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float2 f = Half<T>::unpack(u[q]), g = Half<T>::unpack(v[q]);
            s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
        }
        return s;
    };
    auto sum16 = [](float s) {
#pragma unroll
        for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        return s;
    };
    uint32_t most[2] = {0u, 0u};
    auto larger = [](uint32_t &top, float s) {   // of finite numbers, none negative: their bits are in order
        const uint32_t b = __float_as_uint(s);
        if (b < 0x7f800000u) top = max(top, b);
    };
    auto row = [&](int x0) {   // of 16 threads
        const int x = x0 + (threadIdx.x >> 4), h = hk * group + x % group;
        const int64_t t = t0 + x / group;
        const bool in = x < rows && c < a.width;
        const uint4 o = read(a.out, t, h, in), g = read(a.dout, t, h, in);
        const float s = sum16(dot(o, g));
        if constexpr (WG_P_EXP<T> != 0) larger(most[0], sum16(dot(g, g)));
        if (in && c == 0) {
            const int64_t at = h * a.s.tokens + t;
            delta[at] = s;
            lse2[at] = 1.4426950408889634f * a.lse[at] - WG_P_EXP<T>;
        }
    };
#pragma unroll 1
    for (int x0 = 64 * blockIdx.y; x0 < rows; x0 += 64 * gridDim.y) {
        if (x0 + 64 <= rows) {
#pragma unroll
            for (int i = 0; i < 4; i++) row(x0 + 16 * i);
        } else {
#pragma unroll 1
            for (int x = x0; x < rows; x += 16) row(x);
        }
    }
    if constexpr (WG_P_EXP<T> != 0) {
        for (int x0 = 64 * blockIdx.y; x0 < min(m, 64 * ((int)blockIdx.y + 1)); x0 += 16) {
            const int x = x0 + (threadIdx.x >> 4);
            const uint4 v = read(a.v, t0 + x, hk, x < m && c < a.width);
            larger(most[1], sum16(dot(v, v)));
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            most[i] = __reduce_max_sync(0xffffffffu, most[i]);
            if ((threadIdx.x & 31) == 0 && most[i]) atomicMax(range + 2 * ((int64_t)e.w * a.kv_heads + hk) + i, most[i]);
        }
    }
}

constexpr int WG_COPY = 8, WG_PRODUCTS = 9, WG_THREADS = 320, WG_KEY_BLOCKS = 12;
// Two threads share a row of scores, 64 columns each, and write their 16-bit operands over the first 32 of their own.
struct GradKernel {
    WindowArgs a;
    CUtensorMap mq, mk, mv, mg, m0, m1;   // q, k, v, dout; the outputs: dk and dv, or dq
    float c;                              // scale log2(e)
    int unit, sink_tiles, slots;          // of the cuts of walks over sinks, below
    float *part;                          // the parts' sums: (slots, tiles with sinks, kv_heads, dk and dv, 128, width)
    const float *lse2, *delta, *range;
    int *err;
};

// A tile of keys that holds sinks is seen by the rest of its sequence.  Where its walk is longer than `unit` tiles of queries it is cut into parts of at most
// that many: a CTA each, whose sums window_grad_sinks adds in order.  A sequence's parts lie from slot 2 group (tiles before it) / unit on: of a walk of x
// units, x > 1, there are ceil(x) <= floor(2 x) parts, so that neighbours do not meet and 2 group tiles / unit slots hold all.
struct CutWalk {
    int4 e;                     // {first row, length, first key, sequence}
    int all, part, parts;       // tiles of queries; this one of so many parts
    __device__ __forceinline__ int per() const { return (all + parts - 1) / parts; }
};
__device__ __forceinline__ int walk_parts(int all, int unit) { return (all - 1) / unit + 1; }
// false: the slot holds no part of tile k of keys
__device__ __forceinline__ bool cut_walk(const GradKernel &p, int slot, int k, CutWalk &w) {
    const WindowArgs &a = p.a;
    const int4 *seq = reinterpret_cast<const int4 *>(a.s.table) + seq_of(a.s, 0);
    const int group = a.heads / a.kv_heads;
    auto base = [&](int i) { return 2 * (int64_t)group * seq[i].z / p.unit; };
    int lo = 0, hi = a.s.sequences;   // the last sequence whose slots begin at this one or before
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        (base(mid) <= slot ? lo : hi) = mid;
    }
    const int4 q = seq[lo];
    w.e = make_int4(q.x, q.y, k * SEQ_TILE, lo);
    w.all = (q.w - k) * group;
    if (k >= q.w) return false;
    w.parts = walk_parts(w.all, p.unit);
    w.part = (int)(slot - base(lo));
    return w.parts > 1 && w.part < w.parts;
}

// A CTA has a tile of 128 keys (rows of tensor memory) and walks over tiles of 128 queries (columns).  Of the products of query tile n,
//     S^T = K Q^T (n + 1)  follows  dV += P^T dout (n),     dP^T = V dout^T (n + 1)  follows  dK += dS^T Q (n),
// so that the weights of n + 1 are taken while the second pair runs, and dS while the first does.
template <typename T, int NB>
__global__ void __launch_bounds__(WG_THREADS, 1) window_grad_keys(const __grid_constant__ GradKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 4 + 7];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    __shared__ __align__(16) float lse_s[2][SEQ_TILE], delta_s[2][SEQ_TILE];
    const WindowArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, group = a.heads / a.kv_heads;
    constexpr int stages = NB == 2 ? 2 : 4;
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u, k_tile = smem, v_tile = smem + NB * WF_BLOCK;
    auto q_tile = [&](int s) { return smem + (2 + 2 * s) * NB * WF_BLOCK; };
    auto g_tile = [&](int s) { return smem + (3 + 2 * s) * NB * WF_BLOCK; };
    // the parts of walks that are cut come first, then the tiles whose walk is whole
    const int cut = p.slots * p.sink_tiles * a.kv_heads, hk = ((int)blockIdx.x < cut ? (int)blockIdx.x : (int)blockIdx.x - cut) % a.kv_heads;
    const bool is_part = (int)blockIdx.x < cut;
    CutWalk w;
    if (is_part) {
        if (!cut_walk(p, blockIdx.x / (p.sink_tiles * a.kv_heads), blockIdx.x / a.kv_heads % p.sink_tiles, w)) return;
    } else {
        w.e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_future(a.s, (blockIdx.x - cut) / a.kv_heads)];
    }
    const int4 e = w.e;
    const int key = e.z;
    // queries from the key's own tile on, to the end of the window, or of the sequence where the tile holds sinks
    const int q0 = key / SEQ_TILE, q1 = (key < a.sinks ? e.y - 1 : (int)min((int64_t)e.y - 1, (int64_t)key + SEQ_TILE - 2 + a.window)) / SEQ_TILE;
    const int per_head = q1 - q0 + 1, all = per_head * group;
    if (!is_part && cut && key < a.sinks && walk_parts(all, p.unit) > 1) return;
    const int n0 = is_part ? w.part * w.per() : 0, tiles = is_part ? min(all, n0 + w.per()) - n0 : all;
    if (tiles <= 0) return;

    if (warp == WG_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    if (tid == 0) {
        for (int i = 0; i < 12; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);    // landed, free (by stage); keys landed, S ready, dP ready, all done
        tc::mbar_init(tc::smem_u32(&bars[12]), 256);                              // P written
        tc::mbar_init(tc::smem_u32(&bars[13]), 256);                              // dS written
        tc::mbar_init(tc::smem_u32(&bars[14]), 1);                                // no products in flight
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s, t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[4]), b_k = tc::smem_u32(&bars[8]), b_s = tc::smem_u32(&bars[9]),
                   b_dp = tc::smem_u32(&bars[10]), b_done = tc::smem_u32(&bars[11]), b_p = tc::smem_u32(&bars[12]), b_ds = tc::smem_u32(&bars[13]);
    if (warp == WG_COPY) {
        if (lane == 0) {
            tc::mbar_expect_tx(b_k, 2 * NB * WF_BLOCK);
            for (int k = 0; k < NB; k++) {
                tc::tma_rows(k_tile + k * WF_BLOCK, &p.mk, 64 * k, hk, e.x + key, b_k);
                tc::tma_rows(v_tile + k * WF_BLOCK, &p.mv, 64 * k, hk, e.x + key, b_k);
            }
            int n = 0;
            for (; n < tiles && !gave_up_s; n++) {
                const int s = n % stages, h = hk * group + (n0 + n) / per_head, q = (q0 + (n0 + n) % per_head) * SEQ_TILE;
                if (n >= stages) wait(b_free + 8 * s, (n / stages - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_full + 8 * s, 2 * NB * WF_BLOCK);
                for (int k = 0; k < NB; k++) {
                    tc::tma_rows(q_tile(s) + k * WF_BLOCK, &p.mq, 64 * k, h, e.x + q, b_full + 8 * s);
                    tc::tma_rows(g_tile(s) + k * WF_BLOCK, &p.mg, 64 * k, h, e.x + q, b_full + 8 * s);
                }
            }
            wait.drain(b_k, 0);
            for (int s = 0; s < stages; s++)
                if (n > s) wait.drain(b_full + 8 * s, ((n - 1 - s) / stages) & 1);
        }
    } else if (warp == WG_PRODUCTS) {
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        const uint32_t i_s = tc::idesc_f16(bf, 128, 128, false, false), i_d = tc::idesc_f16(bf, 128, 64 * NB, false, true);
        wait(b_k, 0);
        wait(b_full, 0);
        tc::fence_after_sync();
        if (tc::elect()) {
            tc::product_rows<NB>(t_s, k_tile, q_tile(0), i_s);
            tc::mma_commit(b_s);
            tc::product_rows<NB>(t_dp, v_tile, g_tile(0), i_s);
            tc::mma_commit(b_dp);
        }
        for (int n = 0; n < tiles; n++) {
            const int s = n % stages, sn = (n + 1) % stages;
            const bool more = n + 1 < tiles;
            if (more) wait(b_full + 8 * sn, ((n + 1) / stages) & 1);
            wait(b_p, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_tmem<64>(t_dv, t_s, g_tile(s), i_d, n);
                if (more) {
                    tc::product_rows<NB>(t_s, k_tile, q_tile(sn), i_s);
                    tc::mma_commit(b_s);
                }
            }
            wait(b_ds, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_tmem<64>(t_dk, t_dp, q_tile(s), i_d, n);
                tc::mma_commit(b_free + 8 * s);
                if (more) {
                    tc::product_rows<NB>(t_dp, v_tile, g_tile(sn), i_s);
                    tc::mma_commit(b_dp);
                } else {
                    tc::mma_commit(b_done);
                }
            }
        }
        wait.drain_products(tc::smem_u32(&bars[14]));
    } else {
        // threads r and r + 128 have key row r, half of the queries each
        const int r = tid & 127, half = tid >> 7, j = key + r;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const float times = grad_range<T>(p.range, a.kv_heads, e.w, hk, a.scale).ds;
        const f32x2 cc = pack2(p.c, p.c), ds = pack2(times, times);
        auto row_sum = [&](int n) {   // -lse2 (threads of the first half) or -delta of a query of tile n
            const int h = hk * group + (n0 + n) / per_head, i = (q0 + (n0 + n) % per_head) * SEQ_TILE + r;
            return i < e.y ? (half ? -times : -1.f) * (half ? p.delta : p.lse2)[h * a.s.tokens + e.x + i] : 0.f;
        };
        float next = row_sum(0);
        for (int n = 0; n < tiles; n++) {
            const int q = (q0 + (n0 + n) % per_head) * SEQ_TILE, s = n % stages;
            (half ? delta_s : lse_s)[n & 1][r] = next;
            tc::bar_sync(1, 256);
            if (n + 1 < tiles) next = row_sum(n + 1);
            if (q + SEQ_TILE > e.y) {   // queries of the next sequence: their rows meet no weight, not even a weight of zero
                wait(b_full + 8 * s, (n / stages) & 1);
                wait(b_s, n & 1);
                wait(b_dp, n & 1);
                if (q + r >= e.y) clear_row(half ? g_tile(s) : q_tile(s), r, 0, 8 * NB);
                tc::fence_async_smem();
            }
            // seen: query q + c sees key j if j <= q + c, q + c - j < window or j is a sink, and the query is one
            const bool sink = j < a.sinks;
            const int low = j - q, up = min(sink ? SEQ_TILE - 1 : j - q + a.window - 1, e.y - 1 - q);
            const int i0 = key + 32 * (warp & 3);   // the warp's first key
            const bool whole = i0 + 31 <= q && (q + SEQ_TILE - 1 - i0 < a.window || i0 + 32 <= a.sinks) && q + SEQ_TILE <= e.y;
            wait(b_s, n & 1);
            __syncwarp();
            tc::fence_after_sync();
            float pr[2][32];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t x[32], w[16];
                tc::tmem_ld32(t_s + lanes + 64 * half + 32 * b, x);
                tc::tmem_ld_wait(x);
#pragma unroll
                for (int c = 0; c < 32; c += 4) {   // lse_s and delta_s hold the negatives
                    const ulonglong2 l = *reinterpret_cast<const ulonglong2 *>(&lse_s[n & 1][64 * half + 32 * b + c]);
                    unpack2(fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), cc, l.x), pr[b][c], pr[b][c + 1]);
                    pr[b][c] = ex2_approx(pr[b][c]);
                    pr[b][c + 1] = ex2_approx(pr[b][c + 1]);
                    const f32x2 e2 = fma2(pack2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])), cc, l.y);
                    if (c & 4) exp2_poly<true>(e2, pr[b][c + 2], pr[b][c + 3]);
                    else {
                        unpack2(e2, pr[b][c + 2], pr[b][c + 3]);
                        pr[b][c + 2] = ex2_approx(pr[b][c + 2]);
                        pr[b][c + 3] = ex2_approx(pr[b][c + 3]);
                    }
                }
                if (!whole)
#pragma unroll
                    for (int c = 0; c < 32; c++) {
                        const int at = 64 * half + 32 * b + c;
                        if (at < low || at > up) pr[b][c] = 0.f;
                    }
#pragma unroll
                for (int c = 0; c < 32; c += 2) w[c >> 1] = Half<T>::pack(pr[b][c], pr[b][c + 1]);
                tc::tmem_st16(t_s + lanes + 64 * half + 16 * b, w);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            tc::mbar_arrive(b_p);
            wait(b_dp, n & 1);
            __syncwarp();
            tc::fence_after_sync();
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t x[32], w[16];
                tc::tmem_ld32(t_dp + lanes + 64 * half + 32 * b, x);
                tc::tmem_ld_wait(x);
#pragma unroll
                for (int c = 0; c < 32; c += 4) {
                    const ulonglong2 d = *reinterpret_cast<const ulonglong2 *>(&delta_s[n & 1][64 * half + 32 * b + c]);
                    float y[4];
                    unpack2(mul2(pack2(pr[b][c], pr[b][c + 1]), fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), ds, d.x)), y[0], y[1]);
                    unpack2(mul2(pack2(pr[b][c + 2], pr[b][c + 3]), fma2(pack2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])), ds, d.y)), y[2], y[3]);
                    if (!whole)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const int at = 64 * half + 32 * b + c + k;
                            if (at < low || at > up) y[k] = 0.f;
                        }
                    w[c >> 1] = Half<T>::pack(y[0], y[1]);
                    w[(c >> 1) + 1] = Half<T>::pack(y[2], y[3]);
                }
                tc::tmem_st16(t_dp + lanes + 64 * half + 16 * b, w);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            tc::mbar_arrive(b_ds);
        }
        wait(b_done, 0);
        __syncwarp();
        tc::fence_after_sync();
        if (is_part) {
            float *row = p.part + ((int64_t)blockIdx.x * 2 + half) * SEQ_TILE * a.width + r * a.width;
            for (int q = 0; q < 2 * NB; q++) {
                uint32_t o[32];
                tc::tmem_ld32((half ? t_dv : t_dk) + lanes + 32 * q, o);
                tc::tmem_ld_wait(o);
#pragma unroll
                for (int c = 0; c < 32; c += 4)
                    if (32 * q + c < a.width) *reinterpret_cast<uint4 *>(row + 32 * q + c) = make_uint4(o[c], o[c + 1], o[c + 2], o[c + 3]);
                __syncwarp();
            }
        } else {
            // the first half stages and stores dk over K, the second dv over V
            const uint32_t out = half ? v_tile : k_tile;
            const GradRange range = grad_range<T>(p.range, a.kv_heads, e.w, hk, a.scale);
            const float f = half ? range.out_v : range.out_s;
            for (int q = 0; q < 2 * NB; q++) {
                uint32_t o[32];
                tc::tmem_ld32((half ? t_dv : t_dk) + lanes + 32 * q, o);
                tc::tmem_ld_wait(o);
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint32_t y[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) y[k] = Half<T>::pack(f * __uint_as_float(o[c + 2 * k]), f * __uint_as_float(o[c + 2 * k + 1]));
                    sts16(out + (q >> 1) * WF_BLOCK + tc::swz(r, 4 * (q & 1) + c / 8), y);
                }
            }
            store_rows<128>(half ? p.m1 : p.m0, half ? a.dv : a.dk, out, hk, e.x + key, min(SEQ_TILE, e.y - key), 0, NB, a.width, r, 3 + half);
        }
        if (r == 0) tc::tma_store_wait_all();
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == WG_COPY) tc::tmem_dealloc(tmem, 512);
}

// dk and dv of the tiles of keys whose walk was cut: the parts' sums, in order.  The CTAs of a tile's first part add them.
template <typename T>
__global__ void __launch_bounds__(256) window_grad_sinks(const __grid_constant__ GradKernel p) {
    const WindowArgs &a = p.a;
    const int k = blockIdx.x % p.sink_tiles, slot = blockIdx.x / p.sink_tiles, hk = blockIdx.y;
    CutWalk w;
    if (!cut_walk(p, slot, k, w) || w.part) return;
    const int4 e = w.e;
    const int used = (w.all + w.per() - 1) / w.per(), rows = min(SEQ_TILE, e.y - e.z), half_size = SEQ_TILE * a.width;
    const int64_t stride = (int64_t)p.sink_tiles * a.kv_heads * 2 * half_size;   // from part to part
    const float *sums = p.part + ((int64_t)blockIdx.x * a.kv_heads + hk) * 2 * half_size;
    const GradRange range = grad_range<T>(p.range, a.kv_heads, e.w, hk, a.scale);
    for (int x = blockIdx.z * 256 + threadIdx.x; x < rows * a.width; x += 16 * 256) {   // pairs of entries: dk, then dv
        const int half = 2 * x >= rows * a.width, at = 2 * x - half * rows * a.width, r = at / a.width, c = at % a.width;
        float2 y = make_float2(0.f, 0.f);
        for (int i = 0; i < used; i++) {
            const float2 v = *reinterpret_cast<const float2 *>(sums + i * stride + half * half_size + at);
            y.x += v.x;
            y.y += v.y;
        }
        *reinterpret_cast<uint32_t *>(row_of<T>(half ? a.dv : a.dk, e.x + e.z + r, hk) + c) = Half<T>::pack((half ? range.out_v : range.out_s) * y.x, (half ? range.out_v : range.out_s) * y.y);
    }
}

// A CTA has a tile of 128 queries (rows of tensor memory) and walks over tiles of 128 keys (columns).  S is computed a tile ahead, into one of two
// places in turn; dP (n + 1) and dQ += dS K (n) run while the weights of n + 1 are taken.
template <typename T, int NB>
__global__ void __launch_bounds__(WG_THREADS, 1) window_grad_queries(const __grid_constant__ GradKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 8 + 7];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    const WindowArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, group = a.heads / a.kv_heads;
    constexpr int slots = NB == 2 ? 5 : 8;
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u, q_tile = smem, g_tile = smem + NB * WF_BLOCK;
    auto slot_tile = [&](int s) { return smem + (2 + s) * NB * WF_BLOCK; };
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_past(a.s, blockIdx.x / a.heads)];
    const int h = blockIdx.x % a.heads, hk = h / group, start = e.z;
    const int first = max(0, start - a.window + 1) / SEQ_TILE, sinks = (int)min(((int64_t)a.sinks + SEQ_TILE - 1) / SEQ_TILE, (int64_t)first);
    const int tiles = sinks + start / SEQ_TILE - first + 1;
    auto key_of = [&](int n) { return SEQ_TILE * (n < sinks ? n : first + n - sinks); };

    if (warp == WG_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    if (tid == 0) {
        for (int i = 0; i < 21; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);    // slot landed, free; queries landed, S ready (two), dP ready, all done
        tc::mbar_init(tc::smem_u32(&bars[21]), 256);                              // dS written
        tc::mbar_init(tc::smem_u32(&bars[22]), 1);                                // no products in flight
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s, t_dp = tmem + 256, t_dq = tmem + 384;   // S at tmem and tmem + 128
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[8]), b_q = tc::smem_u32(&bars[16]), b_s = tc::smem_u32(&bars[17]),
                   b_dp = tc::smem_u32(&bars[19]), b_done = tc::smem_u32(&bars[20]), b_ds = tc::smem_u32(&bars[21]);
    if (warp == WG_COPY) {
        if (lane == 0) {
            tc::mbar_expect_tx(b_q, 2 * NB * WF_BLOCK);
            for (int k = 0; k < NB; k++) {
                tc::tma_rows(q_tile + k * WF_BLOCK, &p.mq, 64 * k, h, e.x + start, b_q);
                tc::tma_rows(g_tile + k * WF_BLOCK, &p.mg, 64 * k, h, e.x + start, b_q);
            }
            int x = 0;
            for (; x < 2 * tiles && !gave_up_s; x++) {   // K and V in turn
                const int s = x % slots;
                if (x >= slots) wait(b_free + 8 * s, (x / slots - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_full + 8 * s, NB * WF_BLOCK);
                for (int k = 0; k < NB; k++) tc::tma_rows(slot_tile(s) + k * WF_BLOCK, x & 1 ? &p.mv : &p.mk, 64 * k, hk, e.x + key_of(x >> 1), b_full + 8 * s);
            }
            wait.drain(b_q, 0);
            for (int s = 0; s < slots; s++)
                if (x > s) wait.drain(b_full + 8 * s, ((x - 1 - s) / slots) & 1);
        }
    } else if (warp == WG_PRODUCTS) {
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        const uint32_t i_s = tc::idesc_f16(bf, 128, 128, false, false), i_d = tc::idesc_f16(bf, 128, 64 * NB, false, true);
        auto landed = [&](int x) {
            wait(b_full + 8 * (x % slots), (x / slots) & 1);
            tc::fence_after_sync();
        };
        auto scores = [&](int n) {
            landed(2 * n);
            if (tc::elect()) {
                tc::product_rows<NB>(tmem + 128 * (n & 1), q_tile, slot_tile(2 * n % slots), i_s);
                tc::mma_commit(b_s + 8 * (n & 1));
            }
        };
        auto values = [&](int n) {
            landed(2 * n + 1);
            if (tc::elect()) {
                tc::product_rows<NB>(t_dp, g_tile, slot_tile((2 * n + 1) % slots), i_s);
                tc::mma_commit(b_dp);
                tc::mma_commit(b_free + 8 * ((2 * n + 1) % slots));
            }
        };
        wait(b_q, 0);
        scores(0);
        values(0);
        if (tiles > 1) scores(1);
        for (int n = 0; n < tiles; n++) {
            wait(b_ds, n & 1);
            tc::fence_after_sync();
            if (n + 1 < tiles) values(n + 1);
            if (tc::elect()) {
                tc::product_tmem<64>(t_dq, tmem + 128 * (n & 1), slot_tile(2 * n % slots), i_d, n);
                tc::mma_commit(b_free + 8 * (2 * n % slots));
                if (n + 1 == tiles) tc::mma_commit(b_done);
            }
            if (n + 2 < tiles) scores(n + 2);
        }
        wait.drain_products(tc::smem_u32(&bars[22]));
    } else {
        const int r = tid & 127, half = tid >> 7, i = start + r, i0 = start + 32 * (warp & 3);
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const int64_t at_row = h * a.s.tokens + e.x + i;
        const GradRange range = grad_range<T>(p.range, a.kv_heads, e.w, hk, a.scale);
        const float shift = i < e.y ? -p.lse2[at_row] : 0.f, dl = i < e.y ? -range.ds * p.delta[at_row] : 0.f;
        const f32x2 cc = pack2(p.c, p.c), ss = pack2(shift, shift), ds = pack2(range.ds, range.ds), dd = pack2(dl, dl);
        for (int n = 0; n < tiles; n++) {
            const int key = key_of(n);
            const uint32_t t_s = tmem + 128 * (n & 1);
            const bool whole = key + SEQ_TILE - 1 <= i0 && (i0 + 31 - key < a.window || key + SEQ_TILE <= a.sinks);
            const int up = i - key, low = i - key - a.window, sink = a.sinks - key;   // seen: c <= up and (c > low or c < sink)
            wait(b_s + 8 * (n & 1), (n >> 1) & 1);
            __syncwarp();
            tc::fence_after_sync();
            float pr[2][32];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t x[32];
                tc::tmem_ld32(t_s + lanes + 64 * half + 32 * b, x);
                tc::tmem_ld_wait(x);
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const f32x2 y = fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), cc, ss);
                    if (c % 8 == 6) exp2_poly<true>(y, pr[b][c], pr[b][c + 1]);
                    else {
                        unpack2(y, pr[b][c], pr[b][c + 1]);
                        pr[b][c] = ex2_approx(pr[b][c]);
                        pr[b][c + 1] = ex2_approx(pr[b][c + 1]);
                    }
                }
            }
            if (key + SEQ_TILE > e.y) {   // keys of the next sequence
                const int x = 2 * n, s = x % slots;
                wait(b_full + 8 * s, (x / slots) & 1);
                if (key + r >= e.y) clear_row(slot_tile(s), r, half ? 4 * NB : 0, half ? 8 * NB : 4 * NB);
                tc::fence_async_smem();
            }
            wait(b_dp, n & 1);
            __syncwarp();
            tc::fence_after_sync();
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t x[32], w[16];
                tc::tmem_ld32(t_dp + lanes + 64 * half + 32 * b, x);
                tc::tmem_ld_wait(x);
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float y[2];
                    unpack2(mul2(pack2(pr[b][c], pr[b][c + 1]), fma2(pack2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), ds, dd)), y[0], y[1]);
                    if (!whole)
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const int at = 64 * half + 32 * b + c + k;
                            if (!(at <= up && (at > low || at < sink))) y[k] = 0.f;
                        }
                    w[c >> 1] = Half<T>::pack(y[0], y[1]);
                }
                tc::tmem_st16(t_s + lanes + 64 * half + 16 * b, w);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            tc::mbar_arrive(b_ds);
        }
        wait(b_done, 0);
        __syncwarp();
        tc::fence_after_sync();
        // over Q: the halves take its blocks in turn, at one block half of it each
        for (int q = half * NB; q < (half + 1) * NB; q++) {
            uint32_t o[32];
            tc::tmem_ld32(t_dq + lanes + 32 * q, o);
            tc::tmem_ld_wait(o);
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
                uint32_t y[4];
#pragma unroll
                for (int k = 0; k < 4; k++) y[k] = Half<T>::pack(range.out_s * __uint_as_float(o[c + 2 * k]), range.out_s * __uint_as_float(o[c + 2 * k + 1]));
                sts16(q_tile + (q >> 1) * WF_BLOCK + tc::swz(r, 4 * (q & 1) + c / 8), y);
            }
        }
        store_rows<256>(p.m0, a.dq, q_tile, h, e.x + start, min(SEQ_TILE, e.y - start), 0, NB, a.width, tid, 1);
        if (tid == 0) tc::tma_store_wait_all();
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == WG_COPY) tc::tmem_dealloc(tmem, 512);
}

// Where walks over sinks are cut (CutWalk).  A part is no shorter than the walk of another tile, than 24 tiles of queries, than a sixteenth of the
// longest walk, and than an SM's share of all walks over sinks, halved: where these fill the SMs by themselves they are not cut, and the parts' sums never take
// more than 4 x 148 slots, 78 MB at width 128.  5 packed documents of up to 3000 tokens, window 512, spent 272 us on one walk of 96 tiles, and 68 us' worth of work.
// One of 16384 tokens and 2000 of 64, 32 heads on 8, width 128, window 128, 4 sinks, gradients: 5350 us, some 200 less without sinks; with the longest walk's number of
// parts for every sequence 11000 us and 33.6 GB.
struct GradCuts {
    int unit, sink_tiles;
    int64_t slots;
};
static GradCuts grad_cuts(const f3m_seqs &s, int heads, int kv_heads, int window, int sinks) {
    const int64_t group = heads / kv_heads, longest = ((int64_t)s.longest + SEQ_TILE - 1) / SEQ_TILE, other = std::min(longest, ((int64_t)window + SEQ_TILE - 1) / SEQ_TILE + 1);
    const int64_t ns = ((int64_t)std::min(sinks, s.longest) + SEQ_TILE - 1) / SEQ_TILE, sms = 2 * NUM_SMS_HINT;
    const int64_t share = (s.tiles * group * kv_heads + sms - 1) / sms * ns;
    const int64_t unit = std::max({(int64_t)24, other * group, (longest * group + 15) / 16, share});
    if (ns == 0 || longest * group <= unit) return {0x7fffffff, (int)ns, 0};
    return {(int)unit, (int)ns, 2 * group * s.tiles / unit};
}
static size_t range_floats(const f3m_seqs &s, int kv_heads) { return (2 * (size_t)s.sequences * kv_heads + 3) / 4 * 4; }
static size_t part_floats(const GradCuts &c, int kv_heads, int width) { return (size_t)c.slots * c.sink_tiles * kv_heads * 2 * SEQ_TILE * width; }
size_t window_grad_workspace(const f3m_seqs &s, int heads, int kv_heads, int width, int window, int sinks) {
    const size_t rows = ((size_t)s.tokens * heads + 3) / 4 * 4;
    return (2 * rows + range_floats(s, kv_heads) + part_floats(grad_cuts(s, heads, kv_heads, window, sinks), kv_heads, width)) * sizeof(float);
}

template <typename T>
static void backward_t(const WindowArgs &a, cudaStream_t s) {
    constexpr int type = Half<T>::type, bytes = WF_BLOCKS * WF_BLOCK + 1024;
    const int64_t rows = a.s.tokens * a.heads, n = a.s.tokens;
    F3M_REQUIRE((int64_t)a.s.tiles * a.heads <= 0x7fffffff, F3M_ERR_OVERFLOW, "%lld tokens of %d heads do not fit in 31 bits", (long long)n, a.heads);
    GradKernel p;
    p.a = a;
    p.a.window = std::min(a.window, a.s.longest);   // places and their differences stay within 31 bits
    p.a.sinks = std::min(a.sinks, a.s.longest);
    float *lse2 = a.delta + (rows + 3) / 4 * 4;
    p.lse2 = lse2;
    p.delta = a.delta;
    const GradCuts cuts = grad_cuts(a.s, a.heads, a.kv_heads, a.window, a.sinks);
    p.unit = cuts.unit;
    p.sink_tiles = cuts.sink_tiles;
    p.slots = (int)cuts.slots;
    float *range = lse2 + (rows + 3) / 4 * 4;
    p.range = range;
    p.part = range + range_floats(a.s, a.kv_heads);
    const int64_t parts = cuts.slots * cuts.sink_tiles * a.kv_heads;
    F3M_REQUIRE(a.s.tiles * (int64_t)a.kv_heads + parts <= 0x7fffffff, F3M_ERR_OVERFLOW, "%d tiles of %d heads do not fit in 31 bits", a.s.tiles, a.heads);
    if (WG_P_EXP<T>) F3M_CUDA(cudaMemsetAsync(range, 0, range_floats(a.s, a.kv_heads) * sizeof(float), s));
    const int most_rows = std::min(a.s.longest, SEQ_TILE) * (a.heads / a.kv_heads);
    window_rows_sum<T><<<dim3(a.s.tiles * a.kv_heads, std::min((most_rows + 63) / 64, 65535)), 256, 0, s>>>(a, lse2, a.delta, reinterpret_cast<uint32_t *>(range));
    F3M_LAUNCH_CHECK();
    p.mq = seq_tensor_map(type, a.q, n, a.heads, a.width);
    p.mk = seq_tensor_map(type, a.k, n, a.kv_heads, a.width);
    p.mv = seq_tensor_map(type, a.v, n, a.kv_heads, a.width);
    p.mg = seq_tensor_map(type, a.dout, n, a.heads, a.width);
    p.m0 = seq_tensor_map(type, a.dk, n, a.kv_heads, a.width);
    p.m1 = seq_tensor_map(type, a.dv, n, a.kv_heads, a.width);
    p.c = a.scale * 1.4426950408889634f;
    p.err = seq_error_word();
    constexpr int key_bytes = WG_KEY_BLOCKS * WF_BLOCK + 1024;
    auto keys = a.width <= 64 ? window_grad_keys<T, 1> : window_grad_keys<T, 2>;
    static SharedMemory allowed[2][2];
    allowed[0][a.width > 64].allow(keys, key_bytes);
    keys<<<(unsigned)(parts + a.s.tiles * (int64_t)a.kv_heads), WG_THREADS, key_bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
    if (parts) {
        window_grad_sinks<T><<<dim3(p.slots * p.sink_tiles, a.kv_heads, 16), 256, 0, s>>>(p);
        F3M_LAUNCH_CHECK();
    }
    p.m0 = seq_tensor_map(type, a.dq, n, a.heads, a.width);
    auto queries = a.width <= 64 ? window_grad_queries<T, 1> : window_grad_queries<T, 2>;
    allowed[1][a.width > 64].allow(queries, bytes);
    queries<<<a.s.tiles * a.heads, WG_THREADS, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
}
void window_forward(int type, const WindowArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? forward_t<__nv_bfloat16>(a, s) : forward_t<__half>(a, s); }
void window_backward(int type, const WindowArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? backward_t<__nv_bfloat16>(a, s) : backward_t<__half>(a, s); }

// ---- one new token ----------------------------------------------------------------------------------------------------------
// The cache is read once, by CTAs that each take a part of the keys of one key head for up to 16 query heads that share it; four warps take 16 keys at a
// time in turn.  Memory is the bound, 16 operations a byte at eight heads a key head; the products run on mma.sync (m16n8k16), whose
// fragments come straight from global memory: a contraction does not mind the order of its terms, so lane (g, t) of a warp reads 16 bytes of
// key g, columns 32 s + 8 t .. + 7, and uses them as its terms of two steps; of the values it reads 16 bytes of keys 2t, 2t + 1, 2t + 8, 2t + 9,
// columns 64 f + 8 g .. + 7, and output column n of tile j stands for column 64 f + 8 n + j.  Parts are joined by step_join.
// 32 sequences of up to 16384 tokens, 32 heads on 8, width 128, window 4096: 97-99 us, 4.6 TB/s, 70 % of the measured copy.
// At width 128 three CTAs an SM leave 168 registers a thread, of which 116 bytes are spilled (100 read back): loads of the next keys have no place beside these.
constexpr int ST_THREADS = 128, ST_HEADS = 16;

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (Half<T>::type == F3M_TYPE_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load16(const void *p, bool in) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (in) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// DF: halves of 64 columns
template <typename T, int DF>
__global__ void __launch_bounds__(ST_THREADS, 3) step_keys(StepArgs a) {
    __shared__ float stat[2][4][ST_HEADS];
    __shared__ __align__(16) float sum_s[4][ST_HEADS][64 * DF];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.heads / a.kv_heads, blocks = (group + ST_HEADS - 1) / ST_HEADS, hk = blockIdx.y / blocks, hb = blockIdx.y % blocks;
    const int h0 = hk * group + hb * ST_HEADS, heads = min(ST_HEADS, group - hb * ST_HEADS), part = blockIdx.x;
    const int64_t b = blockIdx.z;
    // the keys seen, numbered without a gap: the sinks before the window, then the window
    const int len = min(max(a.lengths[b], 0), (int)a.capacity), lo = max(0, len - a.window), ns = min(a.sinks, lo), seen = ns + len - lo;
    const int per = ((seen + a.parts - 1) / a.parts + 63) / 64 * 64, v0 = (int)min((int64_t)part * per, (int64_t)seen), v1 = (int)min((int64_t)v0 + per, (int64_t)seen);
    const T *kc = reinterpret_cast<const T *>(a.k.data) + b * a.k_seq + hk * a.k.head_stride, *vc = reinterpret_cast<const T *>(a.v.data) + b * a.v_seq + hk * a.v.head_stride;
    auto key = [&](int v) { return (int64_t)(v < ns ? v : lo + v - ns); };

    uint4 q[2][2 * DF];
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
        for (int s = 0; s < 2 * DF; s++) {
            const int h = g + 8 * r, d = 32 * s + 8 * t;
            q[r][s] = h < heads && d < a.width ? *reinterpret_cast<const uint4 *>(row_of<T>(a.q, b, h0 + h) + d) : make_uint4(0u, 0u, 0u, 0u);
        }
    float o[DF][8][4] = {}, top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    const float c = a.scale * 1.4426950408889634f;
    for (int v = v0 + 16 * warp; v < v1; v += 64) {
        uint4 kf[2][2 * DF], vf[DF][4];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int at = v + 8 * n + g;
            const T *row = kc + key(at) * a.k.token_stride + 8 * t;
#pragma unroll
            for (int s = 0; s < 2 * DF; s++) kf[n][s] = load16(row + 32 * s, at < v1 && 32 * s + 8 * t < a.width);
        }
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int at = v + 8 * (k >> 1) + 2 * t + (k & 1);
            const T *row = vc + key(at) * a.v.token_stride + 8 * g;
#pragma unroll
            for (int f = 0; f < DF; f++) vf[f][k] = load16(row + 64 * f, at < v1 && 64 * f + 8 * g < a.width);
        }
        float x[2][4] = {};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int s = 0; s < 2 * DF; s++) {
                const uint32_t a0[4] = {q[0][s].x, q[1][s].x, q[0][s].y, q[1][s].y}, a1[4] = {q[0][s].z, q[1][s].z, q[0][s].w, q[1][s].w};
                mma_16x8x16<T>(x[n], a0, kf[n][s].x, kf[n][s].y);
                mma_16x8x16<T>(x[n], a1, kf[n][s].z, kf[n][s].w);
            }
        uint32_t w[4];
#pragma unroll
        for (int r = 0; r < 2; r++) {   // heads g and g + 8
            float high = top[r];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    float &y = x[n][2 * r + i];
                    y = v + 8 * n + 2 * t + i < v1 ? y * c : -INFINITY;
                    high = fmaxf(high, y);
                }
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
            if (__any_sync(0xffffffffu, high > top[r])) {
                const float f = ex2_approx(top[r] - high);   // of -inf, where nothing came before: 0
                sum[r] *= f;
                top[r] = high;
#pragma unroll
                for (int k = 0; k < DF; k++)
#pragma unroll
                    for (int j = 0; j < 8; j++) { o[k][j][2 * r] *= f; o[k][j][2 * r + 1] *= f; }
            }
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const float y0 = ex2_approx(x[n][2 * r] - high), y1 = ex2_approx(x[n][2 * r + 1] - high);
                sum[r] += y0 + y1;
                w[2 * n + r] = Half<T>::pack(y0, y1);
            }
        }
#pragma unroll
        for (int f = 0; f < DF; f++) {
            const uint32_t *v0p = reinterpret_cast<const uint32_t *>(&vf[f][0]), *v1p = reinterpret_cast<const uint32_t *>(&vf[f][1]),
                           *v2p = reinterpret_cast<const uint32_t *>(&vf[f][2]), *v3p = reinterpret_cast<const uint32_t *>(&vf[f][3]);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
                mma_16x8x16<T>(o[f][j], w, __byte_perm(v0p[j >> 1], v1p[j >> 1], sel), __byte_perm(v2p[j >> 1], v3p[j >> 1], sel));
            }
        }
    }
    // the warps' sums, scaled to their common maximum
#pragma unroll
    for (int r = 0; r < 2; r++) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
        if (t == 0) { stat[0][warp][g + 8 * r] = top[r]; stat[1][warp][g + 8 * r] = sum[r]; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int h = g + 8 * r;
        const float high = fmaxf(fmaxf(stat[0][0][h], stat[0][1][h]), fmaxf(stat[0][2][h], stat[0][3][h]));
        const float f = top[r] == -INFINITY ? 0.f : ex2_approx(top[r] - high);
#pragma unroll
        for (int k = 0; k < DF; k++)
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int i = 0; i < 2; i++) sum_s[warp][h][64 * k + 8 * (2 * t + i) + j] = f * o[k][j][2 * r + i];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < heads * a.width / 2; x += ST_THREADS) {
        const int h = 2 * x / a.width, d = 2 * x % a.width;
        const float high = fmaxf(fmaxf(stat[0][0][h], stat[0][1][h]), fmaxf(stat[0][2][h], stat[0][3][h]));
        float total = 0.f;
        float2 y = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            if (stat[1][w][h] != 0.f) total += stat[1][w][h] * ex2_approx(stat[0][w][h] - high);   // of a warp without keys: 0
            y.x += sum_s[w][h][d];
            y.y += sum_s[w][h][d + 1];
        }
        if (a.parts == 1) {
            const float inv = total != 0.f ? 1.f / total : 0.f;   // no keys at all: 0; what is not a number stays that
            *reinterpret_cast<uint32_t *>(row_of<T>(a.out, b, h0 + h) + d) = Half<T>::pack(y.x * inv, y.y * inv);
        } else {
            const int64_t row = (b * a.heads + h0 + h) * a.parts + part;
            if (total != 0.f) *reinterpret_cast<float2 *>(a.part + (int64_t)a.n * a.heads * a.parts * 2 + row * a.width + d) = y;
            if (d == 0) *reinterpret_cast<float2 *>(a.part + 2 * row) = make_float2(high, total);
        }
    }
}

// A CTA per (sequence, head): the parts' sums, scaled to their common maximum, in the order of the parts.  A part without keys has a sum of 0, any other
// one of 1 or more, or one that is not a number.
template <typename T>
__global__ void __launch_bounds__(64) step_join(StepArgs a) {
    __shared__ float w_s[256];
    const int64_t b = blockIdx.x / a.heads, row = (int64_t)blockIdx.x * a.parts;
    const int h = blockIdx.x % a.heads, d = 2 * threadIdx.x;
    const float2 *stat = reinterpret_cast<const float2 *>(a.part) + row;
    const float *sums = a.part + (int64_t)a.n * a.heads * a.parts * 2 + row * a.width;
    float high = -INFINITY;
    for (int i = 0; i < a.parts; i++) high = fmaxf(high, stat[i].x);
    for (int i = threadIdx.x; i < a.parts; i += 64) w_s[i] = ex2_approx(stat[i].x - high);
    __syncthreads();
    if (d >= a.width) return;
    float total = 0.f;
    float2 y = make_float2(0.f, 0.f);
    for (int i = 0; i < a.parts; i++) {
        if (stat[i].y == 0.f) continue;   // its sums have not been written
        total += w_s[i] * stat[i].y;
        const float2 x = *reinterpret_cast<const float2 *>(sums + (int64_t)i * a.width + d);
        y.x = fmaf(w_s[i], x.x, y.x);
        y.y = fmaf(w_s[i], x.y, y.y);
    }
    const float inv = total != 0.f ? 1.f / total : 0.f;
    *reinterpret_cast<uint32_t *>(row_of<T>(a.out, b, h) + d) = Half<T>::pack(y.x * inv, y.y * inv);
}

// As many parts as make two waves of CTAs (three to an SM), none below 256 keys; how many keys a sequence has is known on the device only.  32 sequences,
// 8 key heads, 4100 keys: four parts by this rule, 97 us; two take 95, three 113, five 105, six 99.
int window_step_parts(int n, int heads, int kv_heads, int64_t capacity, int window, int sinks) {
    const int64_t most = std::min<int64_t>(capacity, (int64_t)window + sinks), blocks = (heads / kv_heads + ST_HEADS - 1) / ST_HEADS;
    const int64_t ctas = (int64_t)n * kv_heads * blocks, want = (6 * NUM_SMS_HINT + ctas - 1) / ctas;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, (most + 255) / 256, 256}));
}
size_t window_step_part_floats(int n, int heads, int width, int parts) { return parts == 1 ? 0 : (size_t)n * heads * parts * (width + 2); }

template <typename T>
static void step_t(const StepArgs &a, cudaStream_t s) {
    const int blocks = (a.heads / a.kv_heads + ST_HEADS - 1) / ST_HEADS;
    F3M_REQUIRE(a.n <= 65535 && (int64_t)a.kv_heads * blocks <= 65535 && (int64_t)a.n * a.heads <= 0x7fffffff, F3M_ERR_UNSUPPORTED, "%d sequences of %d heads in one call", a.n,
                a.heads);
    const dim3 grid(a.parts, a.kv_heads * blocks, a.n);
    if (a.width <= 64) step_keys<T, 1><<<grid, ST_THREADS, 0, s>>>(a);
    else step_keys<T, 2><<<grid, ST_THREADS, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
    if (a.parts > 1) {
        step_join<T><<<a.n * a.heads, 64, 0, s>>>(a);
        F3M_LAUNCH_CHECK();
    }
}
void window_step(int type, const StepArgs &a, cudaStream_t s) {
    StepArgs b = a;
    b.window = (int)std::min<int64_t>(a.window, std::max<int64_t>(a.capacity, 1));   // numbers of keys stay within 31 bits
    b.sinks = (int)std::min<int64_t>(a.sinks, a.capacity);
    type == F3M_TYPE_BF16 ? step_t<__nv_bfloat16>(b, s) : step_t<__half>(b, s);
}

}  // namespace f3m
