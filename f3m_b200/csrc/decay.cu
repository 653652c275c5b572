// Linear attention with a decay for each head: the recurrence over packed sequences, and one new token.
#include "seq.cuh"

namespace f3m {

__device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    unpack2(v, r.x, r.y);
    return r;
}

// A head's sequences, laid end to end in tiles of 128 tokens, are cut into ranges of equally many tiles; a CTA takes one range and carries the
// state S (width of b x width of c, FP32, in tensor memory) through it.  For a tile of m tokens, with L the triangle of powers of the decay:
//
//     O = use * ( upd * (L o A B^T) C + diag(decay^steps) A S )        near pairs one by one, far ones through the state
//     S = decay^m S + (diag(upd * decay^left) B)^T C                   the state moves on by a tile
//
// All products run on the tensor cores.  Warps 0-3 turn A B^T into the weights (rounded to 16 bits, written over it in tensor memory) and scale the
// rows of A S; warps 4-11 split the scaled rows of B into a sum of 16-bit parts, in place, over A, and over the state's operand: the state is kept
// and returned in FP32, and one rounding of what is added to it would leave it 2^-9 off in bf16.  Two parts lose 2^-17 in bf16, and
// in fp16 2^-23 of rows above 1/4, 2^-25 of smaller ones, whose second part is subnormal (3e-5 of a key of 1e-3); a
// state that is returned takes a third in bf16, one that only serves the tiles behind it does not.  As an operand of A S the state is rounded to
// 16 bits, like the weights.  The tensor cores' FP32 sums round towards zero: a state comes out about 1e-6 off (relative norm), some 0.7e-6 of it short.
//
// What bounds it: tile by tile, the state's way round -- products of the parts, the state read, rounded, scaled, A S, the parts put over what that has
// read.  The arithmetic of the split, A B^T of the next tile, its weights, the outputs and the copies run beside it.
//
// A range that does not begin with a sequence needs the state that the ranges before it leave: decay_states computes what each range
// adds to the state (B and C only), decay_join runs over the ranges, and decay_tiles starts from that.  B and C are then read
// twice, which is the price of using all SMs when there are fewer heads than SMs.
// 65536 tokens, 8 heads, 128 x 128: 262 us = 65 (states) + 13 (join) + 185, 2.0 TB/s of what has to move and 3.1 of what does; 0.33 of the copy rate
// while decay_tiles runs, tensor pipe 27 % busy.
constexpr int DK_COPY = 12, DK_PRODUCTS = 13, DK_THREADS = 32 * 14;   // warps: 0-3 weights and outputs, 4-11 operands, copies, products
constexpr int MAX_RANGES = 3 * NUM_SMS_HINT;
constexpr int DK_AHEAD = 1;                                            // tiles brought into L2 before their stage is free
constexpr int DS_THREADS = 32 * 10;                                   // decay_states: 0-7 operands, copies, products
constexpr int DK_BLOCK = SEQ_TILE * 128;                     // bytes of a block of 64 columns
constexpr int DK_TILES = 14;                                 // blocks of 64 columns in shared memory: the tiles of all stages and the state

struct DecayKernel {
    DecayArgs a;
    CUtensorMap ma, mb, mc;
    int ranges, per_range;      // per_range tiles each
    float *carry;               // (ranges, heads, width of c, width of b): the state behind each range
    int *err;
};

__device__ __forceinline__ int4 tile_at(const DecayArgs &a, int place) {
    return reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, a.reversed ? a.s.tiles - 1 - place : place)];
}
__device__ __forceinline__ bool tile_begins(const DecayArgs &a, const int4 &e) { return a.reversed ? e.z + SEQ_TILE >= e.y : e.z == 0; }
__device__ __forceinline__ bool tile_ends(const DecayArgs &a, const int4 &e) { return a.reversed ? e.z == 0 : e.z + SEQ_TILE >= e.y; }
__device__ __forceinline__ int tile_rows(const int4 &e) { return min(SEQ_TILE, e.y - e.z); }
// tiles of e's sequence before e, in the order of the walk
__device__ __forceinline__ int tiles_before(const DecayArgs &a, const int4 &e) {
    const int i = e.z / SEQ_TILE, n = (e.y + SEQ_TILE - 1) / SEQ_TILE;
    return a.reversed ? n - 1 - i : i;
}

// 16 columns of row j of a state in memory, from column c0 on.  Consecutive threads have consecutive rows: transposed, (width of c, width of b), their
// accesses join, and so the states between ranges lie; row by row a thread takes 16 bytes at a time.
__device__ __forceinline__ void load_state(uint32_t (&r)[16], const float *src, bool transposed, int wb, int wc, int j, int c0) {
#pragma unroll
    for (int c = 0; c < 16; c++) r[c] = 0u;
    if (!src || j >= wb) return;
    if (transposed) {
#pragma unroll
        for (int c = 0; c < 16; c++)
            if (c0 + c < wc) r[c] = __float_as_uint(src[(c0 + c) * wb + j]);
    } else {
#pragma unroll
        for (int c = 0; c < 16; c += 4)
            if (c0 + c < wc) {
                const uint4 v = *reinterpret_cast<const uint4 *>(src + j * wc + c0 + c);
                r[c] = v.x; r[c + 1] = v.y; r[c + 2] = v.z; r[c + 3] = v.w;
            }
    }
}
__device__ __forceinline__ void store_state(const uint32_t (&r)[16], float *dst, bool transposed, int wb, int wc, int j, int c0) {
    if (j >= wb) return;
    if (transposed) {
#pragma unroll
        for (int c = 0; c < 16; c++)
            if (c0 + c < wc) dst[(c0 + c) * wb + j] = __uint_as_float(r[c]);
    } else {
#pragma unroll
        for (int c = 0; c < 16; c += 4)
            if (c0 + c < wc) *reinterpret_cast<uint4 *>(dst + j * wc + c0 + c) = make_uint4(r[c], r[c + 1], r[c + 2], r[c + 3]);
    }
}

// Half of row j of a tile of B, times f, as a sum of 16-bit parts: 16-byte chunks [c0, c0 + N) of its blocks.  The first part takes the row's place,
// the others stay in registers until their places are free.  !in: zeros.
template <typename T, int PARTS, int N>
__device__ __forceinline__ void split_row(uint32_t head, int j, bool in, f32x2 f, int c0, uint32_t (&tail)[N][4], uint32_t (&rest)[N][4]) {
    const f32x2 minus = pack2(-1.f, -1.f);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t at = head + ((c0 + i) >> 3) * DK_BLOCK + tc::swz(j, (c0 + i) & 7);
        uint32_t v[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float2 u = Half<T>::unpack(in ? v[q] : 0u);
            f32x2 x = mul2(pack2(u.x, u.y), f);
            float2 y = unpack2(x);
            v[q] = Half<T>::pack(y.x, y.y);
            y = Half<T>::unpack(v[q]);
            x = fma2(pack2(y.x, y.y), minus, x);
            y = unpack2(x);
            tail[i][q] = Half<T>::pack(y.x, y.y);
            if (PARTS == 3) {
                y = Half<T>::unpack(tail[i][q]);
                y = unpack2(fma2(pack2(y.x, y.y), minus, x));
                rest[i][q] = Half<T>::pack(y.x, y.y);
            }
        }
        sts16(at, v);
    }
}
template <int N>
__device__ __forceinline__ void put_row(uint32_t tile, int j, int c0, const uint32_t (&v)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; i++) sts16(tile + ((c0 + i) >> 3) * DK_BLOCK + tc::swz(j, (c0 + i) & 7), v[i]);
}

template <typename T, int PARTS, int NB>
__global__ void __launch_bounds__(DK_THREADS, 1) decay_tiles(const __grid_constant__ DecayKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 4 + 12];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    const DecayArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, h = blockIdx.x, range = blockIdx.y;
    const int nc = (a.width_c + 63) / 64;
    const int stage_blocks = 2 * NB + nc, stages = min(4, (DK_TILES - max(NB, nc)) / stage_blocks);
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u, state_s = smem + stages * stage_blocks * DK_BLOCK;
    __shared__ __align__(16) float table_s[32];   // decay^(31 - c), from the end decay^c
    const float l2 = log2_decay(a.log_decay[h]);
    const int first = range * p.per_range, tiles = min(a.s.tiles, first + p.per_range) - first;

    if (warp == DK_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    if (tid == 0) {
        for (int i = 0; i < 4; i++) {
            tc::mbar_init(tc::smem_u32(&bars[i]), 1);                                  // landed (by stage)
            tc::mbar_init(tc::smem_u32(&bars[4 + i]), 1);                              // free again
        }
        for (int i = 8; i < 12; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);         // A B^T, A S, state, outputs done
        for (int i = 12; i < 15; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 128);      // weights written, A S scaled, outputs read
        tc::mbar_init(tc::smem_u32(&bars[17]), 1);                                     // A B^T of odd tiles
        tc::mbar_init(tc::smem_u32(&bars[18]), 128);                                   // weights of odd tiles written
        tc::mbar_init(tc::smem_u32(&bars[19]), 1);                                     // no products in flight
        for (int i = 15; i < 17; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 256);      // B split; state ready as operand and in tensor memory
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    if (tid < 32) table_s[tid] = exp2f(l2 * (a.reversed ? tid : 31 - tid));
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s, t_score = tmem, t_out = tmem + 256, t_state = tmem + 384;   // two places for scores, in turn
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[4]), b_score = tc::smem_u32(&bars[8]), b_inter = tc::smem_u32(&bars[9]),
                   b_moved = tc::smem_u32(&bars[10]), b_done = tc::smem_u32(&bars[11]), b_weights = tc::smem_u32(&bars[12]), b_scaled = tc::smem_u32(&bars[13]),
                   b_read = tc::smem_u32(&bars[14]), b_split = tc::smem_u32(&bars[15]), b_state = tc::smem_u32(&bars[16]);
    auto a_tile = [&](int s) { return smem + s * stage_blocks * DK_BLOCK; };
    auto b_tile = [&](int s) { return a_tile(s) + NB * DK_BLOCK; };
    auto c_tile = [&](int s) { return a_tile(s) + 2 * NB * DK_BLOCK; };
    // Scores are two tiles ahead of the weights at times, and the weights of a tile may be there before the products have asked for those of the tile
    // before: a barrier for even tiles and one for odd, each.  A wait names a phase's parity, so no barrier may complete a phase beyond the one that a role
    // may still be waiting for; every other barrier's next phase needs a step of each role that waits for this one.
    auto b_score_of = [&](int n) { return n & 1 ? tc::smem_u32(&bars[17]) : b_score; };
    auto b_weights_of = [&](int n) { return n & 1 ? tc::smem_u32(&bars[18]) : b_weights; };
    auto all_wait = [&](uint32_t bar, uint32_t parity) {   // a whole warp, which stays together for the instructions that need that
        wait(bar, parity);
        __syncwarp();
    };

    if (warp == DK_COPY) {
        // ---- copies ----
        if (lane == 0) {
            // two stages are too few to keep memory busy: tiles further ahead are brought into L2
            auto ahead = [&](int n) {
                if (n >= tiles) return;
                const int4 e = tile_at(a, first + n);
                for (int k = 0; k < NB; k++) {
                    tc::tma_prefetch_rows(&p.ma, 64 * k, h, e.x + e.z);
                    tc::tma_prefetch_rows(&p.mb, 64 * k, h, e.x + e.z);
                }
                for (int k = 0; k < nc; k++) tc::tma_prefetch_rows(&p.mc, 64 * k, h, e.x + e.z);
            };
            int n = 0;
            for (; n < tiles && !gave_up_s; n++) {
                const int s = n % stages;
                const int4 e = tile_at(a, first + n);
                if (n >= stages) wait(b_free + 8 * s, (n / stages - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_full + 8 * s, stage_blocks * DK_BLOCK);
                for (int k = 0; k < NB; k++) {
                    tc::tma_rows(a_tile(s) + k * DK_BLOCK, &p.ma, 64 * k, h, e.x + e.z, b_full + 8 * s);
                    tc::tma_rows(b_tile(s) + k * DK_BLOCK, &p.mb, 64 * k, h, e.x + e.z, b_full + 8 * s);
                }
                for (int k = 0; k < nc; k++) tc::tma_rows(c_tile(s) + k * DK_BLOCK, &p.mc, 64 * k, h, e.x + e.z, b_full + 8 * s);
                if (n + 1 >= stages) ahead(n + DK_AHEAD);
            }
            for (int s = 0; s < stages; s++)   // the last copy into each stage
                if (n > s) wait.drain(b_full + 8 * s, ((n - 1 - s) / stages) & 1);
        }
    } else if (warp == DK_PRODUCTS) {
        // ---- products ----
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        const uint32_t i_score = tc::idesc_f16(bf, 128, 128, false, false), i_rows = tc::idesc_f16(bf, 128, 64 * nc, false, true),
                       i_state = tc::idesc_f16(bf, 128, 64 * nc, true, true);
        auto score = [&](int n) {
            const int s = n % stages;
            wait(b_full + 8 * s, (n / stages) & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_rows<NB>(t_score + 128 * (n & 1), a_tile(s), b_tile(s), i_score);
                tc::mma_commit(b_score_of(n));
            }
        };
        score(0);
        for (int n = 0; n < tiles; n++) {
            const int s = n % stages;
            if (n) wait(b_read, (n - 1) & 1);
            wait(b_state, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_mixed<NB>(t_out, a_tile(s), state_s, i_rows);
                tc::mma_commit(b_inter);
            }
            // the next tile's scores beside the split's last step, if it has landed: the state does not wait for a copy
            const bool more = n + 1 < tiles, early = more && __all_sync(0xffffffffu, tc::mbar_test(b_full + 8 * ((n + 1) % stages), ((n + 1) / stages) & 1));
            if (early) score(n + 1);
            wait(b_split, n & 1);   // also clears the rows of C that belong to another sequence
            tc::fence_after_sync();
            if (tc::elect()) {
#pragma unroll
                for (int part = 0; part < PARTS; part++) tc::product_cols(t_state, part == 0 ? b_tile(s) : part == 1 ? a_tile(s) : state_s, c_tile(s), i_state, 1);
                tc::mma_commit(b_moved);
            }
            wait(b_weights_of(n), (n >> 1) & 1);
            wait(b_scaled, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_tmem(t_out, t_score + 128 * (n & 1), c_tile(s), i_rows, 1);
                tc::mma_commit(b_done);
                tc::mma_commit(b_free + 8 * s);
            }
            if (more && !early) score(n + 1);
        }
        wait.drain_products(tc::smem_u32(&bars[19]));
    } else if (warp < 4) {
        // ---- weights and outputs: thread i has row i ----
        const int i = tid;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        const float coef = a.use * a.upd;
        const bool wide = rows_wide(a.out);
        auto weights = [&](int n, int m) {
            const uint32_t t_s = t_score + 128 * (n & 1) + lanes;
            all_wait(b_score_of(n), (n >> 1) & 1);
            tc::fence_after_sync();
#pragma unroll 1
            for (int cb = 0; cb < 4; cb++) {
                uint32_t w[16];
                const bool near = a.reversed ? cb >= warp : cb <= warp;   // warp-uniform
                if (near) {
                    uint32_t r[32];
                    tc::tmem_ld32(t_s + 32 * cb, r);
                    tc::tmem_ld_wait(r);
                    if (cb != warp && m == SEQ_TILE) {   // off the diagonal: decay^(to the block's edge) times a table
                        const float f = coef * exp2f(l2 * (a.reversed ? 32 * cb - i : i - 32 * cb - 31));
                        const f32x2 ff = pack2(f, f);
                        const ulonglong2 *tab = reinterpret_cast<const ulonglong2 *>(table_s);
#pragma unroll
                        for (int c = 0; c < 32; c += 4) {
                            const ulonglong2 t = tab[c >> 2];
                            float x[4];
                            unpack2(mul2(pack2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), mul2(ff, t.x)), x[0], x[1]);
                            unpack2(mul2(pack2(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), mul2(ff, t.y)), x[2], x[3]);
                            w[c / 2] = Half<T>::pack(x[0], x[1]);
                            w[c / 2 + 1] = Half<T>::pack(x[2], x[3]);
                        }
                    } else {
                        const float from = a.reversed ? (float)(32 * cb - i) : (float)(i - 32 * cb);
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float x[2];
#pragma unroll
                            for (int q = 0; q < 2; q++) {
                                const float apart = a.reversed ? from + (c + q) : from - (c + q);
                                x[q] = coef * __uint_as_float(r[c + q]) * ex2_approx(l2 * apart);
                                if (apart < 0.f || 32 * cb + c + q >= m) x[q] = 0.f;
                            }
                            w[c / 2] = Half<T>::pack(x[0], x[1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 16; c++) w[c] = 0u;
                }
                // columns 16 cb .. of the weights lie over scores that this warp has read
                tc::tmem_st16(t_s + 16 * cb, w);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            tc::mbar_arrive(b_weights_of(n));
        };
        int4 e = tile_at(a, first);
        weights(0, tile_rows(e));
        for (int n = 0; n < tiles; n++) {
            const int m = tile_rows(e);
            const int4 ahead = n + 1 < tiles ? tile_at(a, first + n + 1) : e;
            const float f = a.use * exp2f(l2 * (a.reversed ? max(m - 1 - i, 0) : i + 1));
            all_wait(b_inter, n & 1);
            tc::fence_after_sync();
#pragma unroll 1
            for (int cb = 0; cb < 2 * nc; cb++) {
                uint32_t x[32];
                tc::tmem_ld32(t_out + lanes + 32 * cb, x);
                tc::tmem_ld_wait(x);
#pragma unroll
                for (int c = 0; c < 32; c++) x[c] = __float_as_uint(f * __uint_as_float(x[c]));
                tc::tmem_st32(t_out + lanes + 32 * cb, x);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            tc::mbar_arrive(b_scaled);
            // the next tile's weights now, if its scores are there, else behind the outputs
            const bool now = n + 1 < tiles && __all_sync(0xffffffffu, tc::mbar_test(b_score_of(n + 1), ((n + 1) >> 1) & 1));
            if (now) weights(n + 1, tile_rows(ahead));
            all_wait(b_done, n & 1);
            tc::fence_after_sync();
            uint16_t *row = reinterpret_cast<uint16_t *>(a.out.data) + (int64_t)(e.x + e.z + i) * a.out.token_stride + (int64_t)h * a.out.head_stride;
#pragma unroll 1
            for (int cb = 0; cb < 2 * nc; cb++) {
                uint32_t x[32], w[16];
                tc::tmem_ld32(t_out + lanes + 32 * cb, x);
                tc::tmem_ld_wait(x);
                if (cb + 1 == 2 * nc) {
                    tc::fence_before_sync();
                    tc::mbar_arrive(b_read);
                }
#pragma unroll
                for (int c = 0; c < 16; c++) w[c] = Half<T>::pack(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1]));
                if (i < m) store_row32(row, w, 32 * cb, a.width_c, wide);
                __syncwarp();
            }
            if (n + 1 < tiles && !now) weights(n + 1, tile_rows(ahead));
            e = ahead;
        }
    } else {
        // ---- operands: threads j and j + 128 have row j of B and C, and row j of the state, half each ----
        const int j = tid & 127, half = (tid - 128) >> 7;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const int64_t plane = (int64_t)a.width_b * a.width_c;
        int4 e = tile_at(a, first), gone = e;
        for (int n = 0; n <= tiles; n++) {
            const int m = tile_rows(e), s = n % stages;
            const int4 ahead = n + 1 < tiles ? tile_at(a, first + n + 1) : e;
            uint32_t tail[4 * NB][4], rest[4 * NB][4];
            if (n < tiles) {
                all_wait(b_full + 8 * s, (n / stages) & 1);
                all_wait(b_score_of(n), (n >> 1) & 1);   // B has been read
                const float f = a.upd * exp2f(l2 * (a.reversed ? j + 1 : max(m - 1 - j, 0)));   // rows behind the sequence: a number, to be times 0
                split_row<T, PARTS, 4 * NB>(b_tile(s), j, j < m, pack2(f, f), 4 * NB * half, tail, rest);
                if (j >= m) clear_row(c_tile(s), j, 4 * nc * half, 4 * nc * (half + 1));
            }
            if (n) {
                all_wait(b_moved, (n - 1) & 1);
                tc::fence_after_sync();
                if (a.state_out && tile_ends(a, gone) && 32 * (warp & 3) < a.width_b) {   // whole warps
                    float *dst = a.state_out + ((int64_t)gone.w * a.heads + h) * plane;
#pragma unroll 1
                    for (int cb = 2 * half * nc; cb < 2 * (half + 1) * nc; cb++) {
                        uint32_t r[16];
                        tc::tmem_ld16(t_state + lanes + 16 * cb, r);
                        tc::tmem_ld_wait(r);
                        store_state(r, dst, a.transposed, a.width_b, a.width_c, j, 16 * cb);
                        __syncwarp();
                    }
                }
                if (n == tiles) break;
            }
            // the state before the tile: from tensor memory, or where a sequence or the range begins
            const bool begins = tile_begins(a, e), fresh = begins || n == 0;
            const float scale = exp2f(l2 * m);
            const float *src = nullptr;
            if (begins) {
                if (a.state_in) src = a.state_in + ((int64_t)e.w * a.heads + h) * plane;
            } else if (n == 0) {
                src = p.carry + ((int64_t)(range - 1) * a.heads + h) * plane;
            }
#pragma unroll 1
            for (int cb = 2 * half * nc; cb < 2 * (half + 1) * nc; cb++) {   // 16 columns at a time
                uint32_t r[16];
                if (!fresh) {
                    tc::tmem_ld16(t_state + lanes + 16 * cb, r);
                    tc::tmem_ld_wait(r);
                } else {
                    load_state(r, src, begins ? a.transposed : !a.joined, a.width_b, a.width_c, j, 16 * cb);
                    __syncwarp();
                }
#pragma unroll
                for (int c = 0; c < 16; c += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) w[q] = Half<T>::pack(__uint_as_float(r[c + 2 * q]), __uint_as_float(r[c + 2 * q + 1]));
                    sts16(state_s + (cb >> 2) * DK_BLOCK + tc::swz(j, 2 * (cb & 3) + c / 8), w);
                }
#pragma unroll
                for (int c = 0; c < 16; c++) r[c] = __float_as_uint(scale * __uint_as_float(r[c]));
                tc::tmem_st16(t_state + lanes + 16 * cb, r);
            }
            tc::tmem_st_wait();
            tc::fence_async_smem();
            tc::fence_before_sync();
            tc::mbar_arrive(b_state);
            all_wait(b_inter, n & 1);   // A and the state's operand have been read
            put_row(a_tile(s), j, 4 * NB * half, tail);
            if (PARTS == 3) put_row(state_s, j, 4 * NB * half, rest);
            tc::fence_async_smem();
            tc::mbar_arrive(b_split);
            gone = e;
            e = ahead;
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == DK_COPY) tc::tmem_dealloc(tmem, 512);
}

// What the range adds to the state of the sequence that runs on into the next range, from zero or from where the sequence begins.  The rows
// of B are scaled to the end of the range at once, so that the state gathers in tensor memory without being touched between tiles: splitting a
// tile runs beside the products of the one before.
template <typename T, int PARTS, int NB>
__global__ void __launch_bounds__(DS_THREADS, 1) decay_states(const __grid_constant__ DecayKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 4 + 4];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    const DecayArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, h = blockIdx.x, range = blockIdx.y;
    const int nc = (a.width_c + 63) / 64, stage_blocks = NB + nc, parts_blocks = (PARTS - 1) * NB;
    // a product reads 128 columns of B, with one block of them the block behind it too: what it finds there goes to rows of the state that are not used
    const int stages = min(4, (DK_TILES - parts_blocks - (NB == 1)) / stage_blocks);
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u, parts_s = smem + stages * stage_blocks * DK_BLOCK;
    const float l2 = log2_decay(a.log_decay[h]);
    const int last = min(a.s.tiles, (range + 1) * p.per_range);
    const int4 end = tile_at(a, last - 1);
    if (tile_ends(a, end)) return;
    const int first = max(range * p.per_range, last - 1 - tiles_before(a, end)), tiles = last - first;
    // token behind the range, as its place in the sequence
    const int stop = a.reversed ? end.z : end.z + SEQ_TILE;

    if (warp == 8) tc::tmem_alloc(tc::smem_u32(&tmem_s), 128);
    if (tid == 0) {
        for (int i = 0; i < 8; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);   // landed, free again (by stage)
        tc::mbar_init(tc::smem_u32(&bars[8]), 256);                             // B split
        tc::mbar_init(tc::smem_u32(&bars[9]), 1);                               // tail and rest have been read
        tc::mbar_init(tc::smem_u32(&bars[10]), 1);                              // all done
        tc::mbar_init(tc::smem_u32(&bars[11]), 1);                              // no products in flight
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t t_state = tmem_s;
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[4]), b_split = tc::smem_u32(&bars[8]), b_tails = tc::smem_u32(&bars[9]),
                   b_done = tc::smem_u32(&bars[10]);
    auto b_tile = [&](int s) { return smem + s * stage_blocks * DK_BLOCK; };
    auto c_tile = [&](int s) { return b_tile(s) + NB * DK_BLOCK; };
    if (warp == 8) {
        if (lane == 0) {
            auto ahead = [&](int n) {
                if (n >= tiles) return;
                const int4 e = tile_at(a, first + n);
                for (int k = 0; k < NB; k++) tc::tma_prefetch_rows(&p.mb, 64 * k, h, e.x + e.z);
                for (int k = 0; k < nc; k++) tc::tma_prefetch_rows(&p.mc, 64 * k, h, e.x + e.z);
            };
            int n = 0;
            for (; n < tiles && !gave_up_s; n++) {
                const int s = n % stages;
                const int4 e = tile_at(a, first + n);
                if (n >= stages) wait(b_free + 8 * s, (n / stages - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_full + 8 * s, stage_blocks * DK_BLOCK);
                for (int k = 0; k < NB; k++) tc::tma_rows(b_tile(s) + k * DK_BLOCK, &p.mb, 64 * k, h, e.x + e.z, b_full + 8 * s);
                for (int k = 0; k < nc; k++) tc::tma_rows(c_tile(s) + k * DK_BLOCK, &p.mc, 64 * k, h, e.x + e.z, b_full + 8 * s);
                if (n + 1 >= stages) ahead(n + DK_AHEAD);
            }
            for (int s = 0; s < stages; s++)
                if (n > s) wait.drain(b_full + 8 * s, ((n - 1 - s) / stages) & 1);
        }
    } else if (warp == 9) {
        const uint32_t i_state = tc::idesc_f16(Half<T>::type == F3M_TYPE_BF16, 128, 64 * nc, true, true);
        for (int n = 0; n < tiles; n++) {
            const int s = n % stages;
            wait(b_full + 8 * s, (n / stages) & 1);
            wait(b_split, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
#pragma unroll
                for (int part = PARTS - 1; part >= 0; part--) {
                    tc::product_cols(t_state, part ? parts_s + (part - 1) * NB * DK_BLOCK : b_tile(s), c_tile(s), i_state, n > 0 || part < PARTS - 1);
                    if (part == 1) tc::mma_commit(b_tails);
                }
                tc::mma_commit(b_free + 8 * s);
                if (n + 1 == tiles) tc::mma_commit(b_done);
            }
        }
        wait.drain_products(tc::smem_u32(&bars[11]));
    } else {
        const int j = tid & 127, half = tid >> 7;
        for (int n = 0; n < tiles; n++) {
            const int4 e = tile_at(a, first + n);
            const int m = tile_rows(e), s = n % stages;
            const float f = a.upd * exp2f(l2 * (a.reversed ? e.z + j + 1 - stop : stop - 1 - e.z - j));
            uint32_t tail[4 * NB][4], rest[4 * NB][4];
            wait(b_full + 8 * s, (n / stages) & 1);
            split_row<T, PARTS, 4 * NB>(b_tile(s), j, j < m, pack2(f, f), 4 * NB * half, tail, rest);
            if (n) wait(b_tails, (n - 1) & 1);
            put_row(parts_s, j, 4 * NB * half, tail);
            if (PARTS == 3) put_row(parts_s + NB * DK_BLOCK, j, 4 * NB * half, rest);
            if (j >= m) clear_row(c_tile(s), j, 4 * nc * half, 4 * nc * (half + 1));
            tc::fence_async_smem();
            tc::mbar_arrive(b_split);
        }
        wait(b_done, 0);
        __syncwarp();
        tc::fence_after_sync();
        if (32 * (warp & 3) < a.width_b) {
            const int64_t plane = (int64_t)a.width_b * a.width_c;
            const int4 b = tile_at(a, first);
            const float *src = tile_begins(a, b) && a.state_in ? a.state_in + ((int64_t)b.w * a.heads + h) * plane : nullptr;
            const float f = exp2f(l2 * (a.reversed ? min(b.y, b.z + SEQ_TILE) - stop : stop - b.z));
            float *dst = p.carry + ((int64_t)range * a.heads + h) * plane;
#pragma unroll 1
            for (int cb = 2 * half * nc; cb < 2 * (half + 1) * nc; cb++) {
                uint32_t r[16];
                tc::tmem_ld16(t_state + ((uint32_t)(32 * (warp & 3)) << 16) + 16 * cb, r);
                tc::tmem_ld_wait(r);
                uint32_t b0[16];
                load_state(b0, src, a.transposed, a.width_b, a.width_c, j, 16 * cb);
#pragma unroll
                for (int c = 0; c < 16; c++) r[c] = __float_as_uint(fmaf(f, __uint_as_float(b0[c]), __uint_as_float(r[c])));
                store_state(r, dst, true, a.width_b, a.width_c, j, 16 * cb);
                __syncwarp();
            }
        }
    }
    __syncwarp();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 8) tc::tmem_dealloc(t_state, 128);
}

// Runs over the ranges of a head: where range r is a stretch of one sequence that began before it, the state behind it is what it adds
// plus the state behind range r - 1, decayed over its tokens.
__global__ void __launch_bounds__(128) decay_join(const __grid_constant__ DecayKernel p) {
    const DecayArgs &a = p.a;
    __shared__ float keep_s[MAX_RANGES];   // what range r leaves of the state behind range r - 1; -1: it leaves nothing to the next
    const int h = blockIdx.y, plane = a.width_b * a.width_c, at = 2 * (blockIdx.x * 128 + threadIdx.x);
    const float l2 = log2_decay(a.log_decay[h]);
    for (int r = threadIdx.x; r + 1 < p.ranges; r += 128) {
        const int4 e = tile_at(a, (r + 1) * p.per_range - 1), b = tile_at(a, r * p.per_range);
        const bool through = e.w == b.w && !tile_begins(a, b);
        keep_s[r] = tile_ends(a, e) ? -1.f : through ? exp2f(l2 * (a.reversed ? min(b.y, b.z + SEQ_TILE) - e.z : e.z + tile_rows(e) - b.z)) : 0.f;
    }
    __syncthreads();
    if (at >= plane) return;
    float2 before = make_float2(0.f, 0.f);
    constexpr int AHEAD = 8;
    for (int r0 = 0; r0 + 1 < p.ranges; r0 += AHEAD) {
        float2 x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (r0 + k + 1 < p.ranges && keep_s[r0 + k] >= 0.f) x[k] = *reinterpret_cast<const float2 *>(p.carry + ((int64_t)(r0 + k) * a.heads + h) * plane + at);
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
            if (r0 + k + 1 < p.ranges && keep_s[r0 + k] >= 0.f) {
                const float f = keep_s[r0 + k];
                if (f > 0.f) {
                    x[k].x = fmaf(f, before.x, x[k].x);
                    x[k].y = fmaf(f, before.y, x[k].y);
                    *reinterpret_cast<float2 *>(p.carry + ((int64_t)(r0 + k) * a.heads + h) * plane + at) = x[k];
                }
                before = x[k];
            }
    }
}

// Sequences without tokens hand their state on.
__global__ void __launch_bounds__(256) decay_empty(DecayArgs a) {
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_of(a.s, blockIdx.x)];
    if (e.y) return;
    const int64_t plane = (int64_t)a.width_b * a.width_c * a.heads;
    for (int64_t i = threadIdx.x; i < plane; i += 256) a.state_out[blockIdx.x * plane + i] = a.state_in ? a.state_in[blockIdx.x * plane + i] : 0.f;
}

// How many ranges a head's tiles are cut into.  One CTA of decay_tiles fills an SM.  With one range the SMs without a head idle; with more, B
// and C are read twice, half as much again, and two more launches take as long as some four tiles: the least time of a CTA's tiles, up to three waves.
// 129 tokens of 8 heads: 11.5 us in one range, 13.5 in two.  65536 tokens of 8 heads, the same arrays again and again: 2204 us in one range, on 8 SMs, 236 in 37.
static int decay_ranges(const f3m_seqs &s, int heads) {
    int best = 1;
    float least = 0.f;
    for (int r = 1; r <= s.tiles && (r == 1 || (int64_t)heads * r <= MAX_RANGES); r++) {
        const int64_t ctas = (int64_t)heads * r, waves = (ctas + NUM_SMS_HINT - 1) / NUM_SMS_HINT;
        const int per = (s.tiles + r - 1) / r;
        const float cost = r == 1 ? (float)(waves * per) : 1.5f * (float)(waves * per) + 4.f;
        if (r == 1 || cost < least) { least = cost; best = r; }
    }
    return best;
}
size_t decay_workspace(const f3m_seqs &s, int heads, int width_b, int width_c) {
    const int r = decay_ranges(s, heads);
    return r == 1 ? 0 : (size_t)r * heads * width_b * width_c * sizeof(float);
}

template <typename T, int PARTS, int NB>
static void launch_parts(const DecayKernel &p, cudaStream_t s) {
    constexpr int bytes = DK_TILES * DK_BLOCK + 1024;
    if (p.ranges > 1 && !p.a.joined) {
        static SharedMemory states;
        states.allow(decay_states<T, PARTS, NB>, bytes);
        decay_states<T, PARTS, NB><<<dim3(p.a.heads, p.ranges - 1), DS_THREADS, bytes, s>>>(p);
        F3M_LAUNCH_CHECK();
        decay_join<<<dim3((p.a.width_b * p.a.width_c / 2 + 127) / 128, p.a.heads), 128, 0, s>>>(p);
        F3M_LAUNCH_CHECK();
    }
    static SharedMemory tiles;
    tiles.allow(decay_tiles<T, PARTS, NB>, bytes);
    decay_tiles<T, PARTS, NB><<<dim3(p.a.heads, p.ranges), DK_THREADS, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
}

template <typename T>
static void decay_product_t(const DecayArgs &a, cudaStream_t s) {
    if (a.state_out && a.s.empty) {
        decay_empty<<<a.s.sequences, 256, 0, s>>>(a);
        F3M_LAUNCH_CHECK();
    }
    if (a.s.tiles == 0) return;
    DecayKernel p;
    p.a = a;
    p.ma = seq_tensor_map(Half<T>::type, a.a, a.s.tokens, a.heads, a.width_b);
    p.mb = seq_tensor_map(Half<T>::type, a.b, a.s.tokens, a.heads, a.width_b);
    p.mc = seq_tensor_map(Half<T>::type, a.c, a.s.tokens, a.heads, a.width_c);
    p.ranges = decay_ranges(a.s, a.heads);
    p.per_range = (a.s.tiles + p.ranges - 1) / p.ranges;
    p.ranges = (a.s.tiles + p.per_range - 1) / p.per_range;
    p.carry = (float *)a.ws;
    p.err = seq_error_word();
    // a state that is returned in FP32 takes three parts of bf16
    if constexpr (Half<T>::type == F3M_TYPE_BF16) {
        if (a.state_out) return a.width_b <= 64 ? launch_parts<T, 3, 1>(p, s) : launch_parts<T, 3, 2>(p, s);
    }
    a.width_b <= 64 ? launch_parts<T, 2, 1>(p, s) : launch_parts<T, 2, 2>(p, s);
}
void decay_product(int type, const DecayArgs &a, cudaStream_t s) { type == F3M_TYPE_BF16 ? decay_product_t<__nv_bfloat16>(a, s) : decay_product_t<__half>(a, s); }

// A CTA per (sequence, head): 32 threads across the columns, four each, 8 rows of threads down the state.  The state is read and written
// once, 16 bytes a thread, and that is all the time there is: 64 sequences, 32 heads, 128 x 128 in 45 us, 6.0 TB/s, 92 % of the measured copy.
template <typename T>
__global__ void __launch_bounds__(256) decay_step_kernel(int heads, int wk, int wv, const float *log_decay, float scale, f3m_rows q, f3m_rows k,
                                                         f3m_rows v, float *state, f3m_rows out) {
    __shared__ float qs[F3M_MAX_WIDTH], ks[F3M_MAX_WIDTH];
    __shared__ float4 part[8][32];
    const int64_t n = blockIdx.x / heads;
    const int h = blockIdx.x % heads, t = threadIdx.x, col = 4 * (t & 31), r0 = t >> 5;
    const float decay = exp2f(log2_decay(log_decay[h]));
    float4 *S = reinterpret_cast<float4 *>(state + (int64_t)blockIdx.x * wk * wv);
    float4 x[16];
    const bool in = col < wv;
#pragma unroll
    for (int r = 0; r < 16; r++)
        if (in && r0 + 8 * r < wk) x[r] = __ldcs(&S[((r0 + 8 * r) * wv + col) >> 2]);
    if (t < wk) {
        qs[t] = scale * (float)(reinterpret_cast<const T *>(q.data)[n * q.token_stride + h * q.head_stride + t]);
        ks[t] = (float)(reinterpret_cast<const T *>(k.data)[n * k.token_stride + h * k.head_stride + t]);
    }
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in) {
        const uint2 w = *reinterpret_cast<const uint2 *>(reinterpret_cast<const T *>(v.data) + n * v.token_stride + h * v.head_stride + col);
        const float2 lo = Half<T>::unpack(w.x), hi = Half<T>::unpack(w.y);
        c = make_float4(lo.x, lo.y, hi.x, hi.y);
    }
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int d = r0 + 8 * r;
        if (in && d < wk) {
            const float kd = ks[d], qd = qs[d];
            x[r].x = fmaf(kd, c.x, decay * x[r].x); x[r].y = fmaf(kd, c.y, decay * x[r].y);
            x[r].z = fmaf(kd, c.z, decay * x[r].z); x[r].w = fmaf(kd, c.w, decay * x[r].w);
            o.x = fmaf(qd, x[r].x, o.x); o.y = fmaf(qd, x[r].y, o.y); o.z = fmaf(qd, x[r].z, o.z); o.w = fmaf(qd, x[r].w, o.w);
            __stcs(&S[(d * wv + col) >> 2], x[r]);
        }
    }
    part[r0][t & 31] = o;
    __syncthreads();
    if (t < 32 && in) {
        for (int r = 1; r < 8; r++) {
            const float4 y = part[r][t];
            o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
        }
        *reinterpret_cast<uint2 *>(reinterpret_cast<T *>(out.data) + n * out.token_stride + h * out.head_stride + col) = make_uint2(Half<T>::pack(o.x, o.y), Half<T>::pack(o.z, o.w));
    }
}

void decay_step(int type, int n, int heads, int wk, int wv, const float *log_decay, float scale, const f3m_rows &q, const f3m_rows &k, const f3m_rows &v,
                float *state, const f3m_rows &out, cudaStream_t s) {
    F3M_REQUIRE((int64_t)n * heads <= 0x7fffffff, F3M_ERR_OVERFLOW, "%d sequences of %d heads do not fit in 31 bits", n, heads);
    if (type == F3M_TYPE_BF16) decay_step_kernel<__nv_bfloat16><<<n * heads, 256, 0, s>>>(heads, wk, wv, log_decay, scale, q, k, v, state, out);
    else decay_step_kernel<__half><<<n * heads, 256, 0, s>>>(heads, wk, wv, log_decay, scale, q, k, v, state, out);
    F3M_LAUNCH_CHECK();
}

}  // namespace f3m
