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
// All products run on the tensor cores.  While warps 0-3 turn A B^T into the weights (rounded to 16 bits, written over it in tensor memory),
// warps 4-11 split the scaled rows of B into a sum of 16-bit parts, in place, over A, and over the state's operand: the state is kept and returned
// in FP32, and one rounding of what is added to it would leave it 2^-9 off in bf16.  Two parts lose 2^-17 (bf16) or 2^-23 (fp16); a state that is
// returned takes a third in bf16, one that only serves the tiles behind it does not.  As an operand of A S the state is rounded to 16
// bits, like the weights.
//
// What bounds it: tile by tile, the state's way round -- parts written, their products, the state read, rounded and scaled, A S, parts of the next
// tile.  A B^T, the weights, their product and the outputs run beside it, and so do the copies of the next tile.
//
// A range that does not begin with a sequence needs the state that the ranges before it leave: decay_states computes what each range
// adds to the state (B and C only), decay_join runs over the ranges, and decay_tiles starts from that.  B and C are then read
// twice, which is the price of using all SMs when there are fewer heads than SMs.
constexpr int DK_COPY = 12, DK_PRODUCTS = 13, DK_THREADS = 32 * 14;   // warps: 0-3 weights and outputs, 4-11 operands, copies, products
constexpr int DS_THREADS = 32 * 10;                                   // decay_states: 0-7 operands, copies, products
constexpr int DK_BLOCK = SEQ_TILE * 128;                     // bytes of a block of 64 columns
constexpr int DK_TILES = 14;                                 // blocks of 64 columns in shared memory: the tiles of all stages and the state

struct DecayKernel {
    DecayArgs a;
    CUtensorMap ma, mb, mc, mo;
    int ranges, per_range;      // per_range tiles each
    float *carry;               // (ranges, heads, width of b, width of c): the state behind each range
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

// 32 columns of row j of a state, from column c0 on
__device__ __forceinline__ void state_row(const uint32_t (&r)[32], float *dst, bool transposed, int wb, int wc, int j, int c0) {
    if (transposed) {
#pragma unroll
        for (int c = 0; c < 32; c++)
            if (j < wb && c0 + c < wc) dst[(int64_t)(c0 + c) * wb + j] = __uint_as_float(r[c]);
    } else {
#pragma unroll
        for (int c = 0; c < 32; c += 4)
            if (j < wb && c0 + c < wc) *reinterpret_cast<uint4 *>(dst + (int64_t)j * wc + c0 + c) = make_uint4(r[c], r[c + 1], r[c + 2], r[c + 3]);
    }
}
// Row j of a tile of B, times f, as a sum of 16-bit parts: 16-byte chunks [c0, c1) of its blocks; the first part stays in place.  j >= rows: zeros.
template <typename T, int PARTS>
__device__ __forceinline__ void split_rows(uint32_t head, uint32_t tail, uint32_t rest, int j, bool in, f32x2 f, int c0, int c1) {
    const f32x2 minus = pack2(-1.f, -1.f);
#pragma unroll 2
    for (int i = c0; i < c1; i++) {
        const uint32_t at = (i >> 3) * DK_BLOCK + tc::swz(j, i & 7);
        uint32_t v[4], w[4], z[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(head + at) : "memory");
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float2 u = Half<T>::unpack(in ? v[q] : 0u);
            f32x2 x = mul2(pack2(u.x, u.y), f);
            float2 y = unpack2(x);
            v[q] = Half<T>::pack(y.x, y.y);
            y = Half<T>::unpack(v[q]);
            x = fma2(pack2(y.x, y.y), minus, x);
            y = unpack2(x);
            w[q] = Half<T>::pack(y.x, y.y);
            if (PARTS == 3) {
                y = Half<T>::unpack(w[q]);
                y = unpack2(fma2(pack2(y.x, y.y), minus, x));
                z[q] = Half<T>::pack(y.x, y.y);
            }
        }
        sts16(head + at, v);
        sts16(tail + at, w);
        if (PARTS == 3) sts16(rest + at, z);
    }
}
template <typename T, int PARTS, int NB>
__global__ void __launch_bounds__(DK_THREADS, 1) decay_tiles(const __grid_constant__ DecayKernel p) {
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[2 * 4 + 8];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    __shared__ __align__(16) float pw[32], pr[32];   // decay^n, decay^(31 - n)
    const DecayArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, h = blockIdx.y;
    const int nc = (a.width_c + 63) / 64;
    const int stage_blocks = 2 * NB + nc, stages = min(4, (DK_TILES - max(NB, nc)) / stage_blocks);
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u, state_s = smem + stages * stage_blocks * DK_BLOCK;
    const float l2 = log2_decay(a.log_decay[h]);
    const int first = blockIdx.x * p.per_range, tiles = min(a.s.tiles, first + p.per_range) - first;

    if (warp == DK_COPY) tc::tmem_alloc(tc::smem_u32(&tmem_s), 512);
    if (tid == 0) {
        for (int i = 0; i < 4; i++) {
            tc::mbar_init(tc::smem_u32(&bars[i]), 1);                                  // landed (by stage)
            tc::mbar_init(tc::smem_u32(&bars[4 + i]), 2);                              // free again: products done, outputs on their way
        }
        tc::mbar_init(tc::smem_u32(&bars[8]), 1);                                      // A B^T done
        tc::mbar_init(tc::smem_u32(&bars[9]), 1);                                      // A S done
        tc::mbar_init(tc::smem_u32(&bars[10]), 1);                                     // state done
        tc::mbar_init(tc::smem_u32(&bars[11]), 1);                                     // outputs done
        tc::mbar_init(tc::smem_u32(&bars[12]), 128);                                   // weights written
        tc::mbar_init(tc::smem_u32(&bars[13]), 256);                                   // B split
        tc::mbar_init(tc::smem_u32(&bars[14]), 256);                                   // state ready as operand and in tensor memory
        tc::mbar_init(tc::smem_u32(&bars[15]), 128);                                   // outputs read
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    if (tid < 32) {
        pw[tid] = exp2f(l2 * tid);
        pr[tid] = exp2f(l2 * (31 - tid));
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const Waits wait{&gave_up_s, p.err};
    const uint32_t tmem = tmem_s, t_score = tmem, t_inter = tmem + 128, t_intra = tmem + 256, t_state = tmem + 384;
    const uint32_t b_full = tc::smem_u32(&bars[0]), b_free = tc::smem_u32(&bars[4]), b_score = tc::smem_u32(&bars[8]), b_inter = tc::smem_u32(&bars[9]),
                   b_moved = tc::smem_u32(&bars[10]), b_done = tc::smem_u32(&bars[11]), b_weights = tc::smem_u32(&bars[12]), b_split = tc::smem_u32(&bars[13]),
                   b_state = tc::smem_u32(&bars[14]), b_read = tc::smem_u32(&bars[15]);
    auto a_tile = [&](int s) { return smem + s * stage_blocks * DK_BLOCK; };
    auto b_tile = [&](int s) { return a_tile(s) + NB * DK_BLOCK; };
    auto c_tile = [&](int s) { return a_tile(s) + 2 * NB * DK_BLOCK; };
    auto all_wait = [&](uint32_t bar, uint32_t parity) {   // a whole warp, which stays together for the instructions that need that
        wait(bar, parity);
        __syncwarp();
    };

    if (warp == DK_COPY) {
        // ---- copies ----
        if (lane == 0) {
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
            }
            for (int s = 0; s < stages; s++)   // the last copy into each stage
                if (n > s) wait.drain(b_full + 8 * s, ((n - 1 - s) / stages) & 1);
        }
    } else if (warp == DK_PRODUCTS) {
        // ---- products ----
        constexpr bool bf = Half<T>::type == F3M_TYPE_BF16;
        const uint32_t i_score = tc::idesc_f16(bf, 128, 128, false, false), i_rows = tc::idesc_f16(bf, 128, 64 * nc, false, true),
                       i_state = tc::idesc_f16(bf, 128, 64 * nc, true, true);
        for (int n = 0; n < tiles; n++) {
            const int s = n % stages;
            wait(b_full + 8 * s, (n / stages) & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_rows<NB>(t_score, a_tile(s), b_tile(s), i_score);
                tc::mma_commit(b_score);
            }
            if (n) wait(b_read, (n - 1) & 1);
            wait(b_state, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_mixed<NB>(t_inter, a_tile(s), state_s, i_rows);
                tc::mma_commit(b_inter);
            }
            wait(b_split, n & 1);   // also clears the rows of C that belong to another sequence
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_cols<true>(t_state, b_tile(s), c_tile(s), i_state);
                tc::product_cols<true>(t_state, a_tile(s), c_tile(s), i_state);
                if (PARTS == 3) tc::product_cols<true>(t_state, state_s, c_tile(s), i_state);
                tc::mma_commit(b_moved);
            }
            wait(b_weights, n & 1);
            tc::fence_after_sync();
            if (tc::elect()) {
                tc::product_tmem<false>(t_intra, t_score, c_tile(s), i_rows);
                tc::mma_commit(b_done);
                tc::mma_commit(b_free + 8 * s);
            }
        }
    } else if (warp < 4) {
        // ---- weights and outputs: thread i has row i ----
        const int i = tid;
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        const float coef = a.use * a.upd;
        for (int n = 0; n < tiles; n++) {
            const int4 e = tile_at(a, first + n);
            const int m = tile_rows(e), s = n % stages;
            all_wait(b_score, n & 1);
            tc::fence_after_sync();
#pragma unroll 1
            for (int cb = 0; cb < 4; cb++) {
                uint32_t w[16];
                const bool near = a.reversed ? cb >= warp : cb <= warp;   // warp-uniform
                if (near) {
                    uint32_t r[32];
                    tc::tmem_ld32(t_score + lanes + 32 * cb, r);
                    tc::tmem_ld_wait(r);
                    if (cb == warp) {
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float x[2];
#pragma unroll
                            for (int q = 0; q < 2; q++) {
                                const int apart = a.reversed ? c + q - lane : lane - c - q;
                                x[q] = apart >= 0 && 32 * cb + c + q < m ? __uint_as_float(r[c + q]) * (coef * pw[max(apart, 0)]) : 0.f;
                            }
                            w[c / 2] = Half<T>::pack(x[0], x[1]);
                        }
                    } else {
                        const float f = coef * exp2f(l2 * (a.reversed ? 32 * cb - i : i - 32 * cb - 31));
                        const float *tab = a.reversed ? pw : pr;
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const float2 t = *reinterpret_cast<const float2 *>(tab + c);
                            const float x0 = __uint_as_float(r[c]) * (f * t.x), x1 = __uint_as_float(r[c + 1]) * (f * t.y);
                            w[c / 2] = Half<T>::pack(32 * cb + c < m ? x0 : 0.f, 32 * cb + c + 1 < m ? x1 : 0.f);
                        }
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 16; c++) w[c] = 0u;
                }
                // columns 16 cb .. of the weights lie over scores that this warp has read
                tc::tmem_st16(t_score + lanes + 16 * cb, w);
            }
            tc::tmem_st_wait();
            tc::fence_before_sync();
            tc::mbar_arrive(b_weights);

            all_wait(b_done, n & 1);
            tc::fence_after_sync();
            // the outputs go over C, which has been read, and leave from there
            const float f = a.use * exp2f(l2 * (a.reversed ? m - 1 - i : i + 1));
#pragma unroll 1
            for (int cb = 0; cb < 2 * nc; cb++) {
                uint32_t x[32], y[32];
                tc::tmem_ld32(t_inter + lanes + 32 * cb, x);
                tc::tmem_ld32(t_intra + lanes + 32 * cb, y);
                tc::tmem_ld_wait(x);
                tc::tmem_ld_wait(y);
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        w[q] = Half<T>::pack(fmaf(f, __uint_as_float(x[c + 2 * q]), __uint_as_float(y[c + 2 * q])),
                                             fmaf(f, __uint_as_float(x[c + 2 * q + 1]), __uint_as_float(y[c + 2 * q + 1])));
                    sts16(c_tile(s) + (cb >> 1) * DK_BLOCK + tc::swz(i, 4 * (cb & 1) + c / 8), w);
                }
            }
            tc::fence_before_sync();
            tc::mbar_arrive(b_read);
            store_rows<128>(p.mo, a.out, c_tile(s), h, e.x + e.z, m, 0, nc, a.width_c, i, 1);
            if (i == 0) tc::mbar_arrive(b_free + 8 * s);
        }
        if (i == 0) tc::tma_store_wait_all();
    } else if (warp < DK_COPY) {
        // ---- operands: threads j and j + 128 have row j of B and C, and row j of the state, half each ----
        const int j = tid & 127, half = (tid - 128) >> 7;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const int64_t plane = (int64_t)a.width_b * a.width_c;
        int4 e = tile_at(a, first);
        for (int n = 0; n < tiles; n++) {
            const int m = tile_rows(e), s = n % stages;
            const int4 ahead = n + 1 < tiles ? tile_at(a, first + n + 1) : e;
            // the state before the tile: from tensor memory, or where a sequence or the range begins
            const bool begins = tile_begins(a, e), fresh = begins || n == 0;
            const float scale = exp2f(l2 * m);
            const float *src = nullptr;
            if (begins) {
                if (a.state_in) src = a.state_in + ((int64_t)e.w * a.heads + h) * plane;
            } else if (n == 0) {
                src = p.carry + ((int64_t)(blockIdx.x - 1) * a.heads + h) * plane;
            }
            const bool turned = begins && a.transposed;
#pragma unroll 1
            for (int cb = half * nc; cb < (half + 1) * nc; cb++) {
                uint32_t r[32];
                if (!fresh) {
                    tc::tmem_ld32(t_state + lanes + 32 * cb, r);
                    tc::tmem_ld_wait(r);
                } else {
#pragma unroll
                    for (int c = 0; c < 32; c++) r[c] = 0u;
                    if (src && j < a.width_b) {
                        if (turned) {
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (32 * cb + c < a.width_c) r[c] = __float_as_uint(src[(int64_t)(32 * cb + c) * a.width_b + j]);
                        } else {
#pragma unroll
                            for (int c = 0; c < 32; c += 4)
                                if (32 * cb + c < a.width_c) {
                                    const uint4 v = *reinterpret_cast<const uint4 *>(src + (int64_t)j * a.width_c + 32 * cb + c);
                                    r[c] = v.x; r[c + 1] = v.y; r[c + 2] = v.z; r[c + 3] = v.w;
                                }
                        }
                    }
                }
                const uint32_t row = state_s + (cb >> 1) * DK_BLOCK;
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int q = 0; q < 4; q++) w[q] = Half<T>::pack(__uint_as_float(r[c + 2 * q]), __uint_as_float(r[c + 2 * q + 1]));
                    sts16(row + tc::swz(j, 4 * (cb & 1) + c / 8), w);
                }
#pragma unroll
                for (int c = 0; c < 32; c++) r[c] = __float_as_uint(scale * __uint_as_float(r[c]));
                __syncwarp();
                tc::tmem_st32(t_state + lanes + 32 * cb, r);
            }
            tc::tmem_st_wait();
            tc::fence_async_smem();
            tc::fence_before_sync();
            tc::mbar_arrive(b_state);

            all_wait(b_full + 8 * s, (n / stages) & 1);
            all_wait(b_inter, n & 1);   // A, B and the state's operand have been read
            const float f = a.upd * exp2f(l2 * (a.reversed ? j + 1 : max(m - 1 - j, 0)));   // rows behind the sequence: a number, to be times 0
            split_rows<T, PARTS>(b_tile(s), a_tile(s), state_s, j, j < m, pack2(f, f), 4 * NB * half, 4 * NB * (half + 1));
            if (j >= m) clear_row(c_tile(s), j, 4 * nc * half, 4 * nc * (half + 1));
            tc::fence_async_smem();
            tc::mbar_arrive(b_split);
            all_wait(b_moved, n & 1);
            tc::fence_after_sync();
            if (a.state_out && tile_ends(a, e) && 32 * (warp & 3) < a.width_b) {   // whole warps
                float *dst = a.state_out + ((int64_t)e.w * a.heads + h) * plane;
#pragma unroll 1
                for (int cb = half * nc; cb < (half + 1) * nc; cb++) {
                    uint32_t r[32];
                    tc::tmem_ld32(t_state + lanes + 32 * cb, r);
                    tc::tmem_ld_wait(r);
                    state_row(r, dst, a.transposed, a.width_b, a.width_c, j, 32 * cb);
                    __syncwarp();
                }
            }
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
    __shared__ __align__(8) uint64_t bars[2 * 4 + 3];
    __shared__ uint32_t tmem_s;
    __shared__ int gave_up_s;
    const DecayArgs &a = p.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, h = blockIdx.y;
    const int nc = (a.width_c + 63) / 64, stage_blocks = NB + nc, parts_blocks = (PARTS - 1) * NB;
    // a product reads 128 columns of B, with one block of them the block behind it too: what it finds there goes to rows of the state that are not used
    const int stages = min(4, (DK_TILES - parts_blocks - (NB == 1)) / stage_blocks);
    const uint32_t smem = (tc::smem_u32(raw) + 1023) & ~1023u, parts_s = smem + stages * stage_blocks * DK_BLOCK;
    const float l2 = log2_decay(a.log_decay[h]);
    const int last = min(a.s.tiles, (int)(blockIdx.x + 1) * p.per_range);
    const int4 end = tile_at(a, last - 1);
    if (tile_ends(a, end)) return;
    const int first = max((int)blockIdx.x * p.per_range, last - 1 - tiles_before(a, end)), tiles = last - first;
    // token behind the range, as its place in the sequence
    const int stop = a.reversed ? end.z : end.z + SEQ_TILE;

    if (warp == 8) tc::tmem_alloc(tc::smem_u32(&tmem_s), 128);
    if (tid == 0) {
        for (int i = 0; i < 8; i++) tc::mbar_init(tc::smem_u32(&bars[i]), 1);   // landed, free again (by stage)
        tc::mbar_init(tc::smem_u32(&bars[8]), 256);                             // B split
        tc::mbar_init(tc::smem_u32(&bars[9]), 1);                               // tail and rest have been read
        tc::mbar_init(tc::smem_u32(&bars[10]), 1);                              // all done
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
            int n = 0;
            for (; n < tiles && !gave_up_s; n++) {
                const int s = n % stages;
                const int4 e = tile_at(a, first + n);
                if (n >= stages) wait(b_free + 8 * s, (n / stages - 1) & 1);
                if (gave_up_s) break;
                tc::mbar_expect_tx(b_full + 8 * s, stage_blocks * DK_BLOCK);
                for (int k = 0; k < NB; k++) tc::tma_rows(b_tile(s) + k * DK_BLOCK, &p.mb, 64 * k, h, e.x + e.z, b_full + 8 * s);
                for (int k = 0; k < nc; k++) tc::tma_rows(c_tile(s) + k * DK_BLOCK, &p.mc, 64 * k, h, e.x + e.z, b_full + 8 * s);
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
                const uint32_t last_part = parts_s + (PARTS - 2) * NB * DK_BLOCK;
                if (n) tc::product_cols<true>(t_state, last_part, c_tile(s), i_state);
                else tc::product_cols<false>(t_state, last_part, c_tile(s), i_state);
                if (PARTS == 3) tc::product_cols<true>(t_state, parts_s, c_tile(s), i_state);
                tc::mma_commit(b_tails);
                tc::product_cols<true>(t_state, b_tile(s), c_tile(s), i_state);
                tc::mma_commit(b_free + 8 * s);
                if (n + 1 == tiles) tc::mma_commit(b_done);
            }
        }
    } else {
        const int j = tid & 127, half = tid >> 7;
        for (int n = 0; n < tiles; n++) {
            const int4 e = tile_at(a, first + n);
            const int m = tile_rows(e), s = n % stages;
            const float f = a.upd * exp2f(l2 * (a.reversed ? e.z + j + 1 - stop : stop - 1 - e.z - j));
            wait(b_full + 8 * s, (n / stages) & 1);
            if (n) wait(b_tails, (n - 1) & 1);
            split_rows<T, PARTS>(b_tile(s), parts_s, parts_s + NB * DK_BLOCK, j, j < m, pack2(f, f), 4 * NB * half, 4 * NB * (half + 1));
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
            float *dst = p.carry + ((int64_t)blockIdx.x * a.heads + h) * plane;
#pragma unroll 1
            for (int cb = half * nc; cb < (half + 1) * nc; cb++) {
                uint32_t r[32];
                tc::tmem_ld32(t_state + ((uint32_t)(32 * (warp & 3)) << 16) + 32 * cb, r);
                tc::tmem_ld_wait(r);
                if (src && j < a.width_b)
#pragma unroll
                    for (int c = 0; c < 32; c++)
                        if (32 * cb + c < a.width_c)
                            r[c] = __float_as_uint(fmaf(f, src[a.transposed ? (int64_t)(32 * cb + c) * a.width_b + j : (int64_t)j * a.width_c + 32 * cb + c], __uint_as_float(r[c])));
                state_row(r, dst, false, a.width_b, a.width_c, j, 32 * cb);
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
__global__ void __launch_bounds__(256) decay_join(const __grid_constant__ DecayKernel p) {
    const DecayArgs &a = p.a;
    const int h = blockIdx.y, plane = a.width_b * a.width_c, at = 4 * (blockIdx.x * 256 + threadIdx.x);
    const float l2 = log2_decay(a.log_decay[h]);
    float4 before = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int r = 0; r + 1 < p.ranges; r++) {
        const int last = (r + 1) * p.per_range;
        const int4 e = tile_at(a, last - 1), b = tile_at(a, r * p.per_range);
        if (tile_ends(a, e) || at >= plane) continue;
        float4 *mine = reinterpret_cast<float4 *>(p.carry + ((int64_t)r * a.heads + h) * plane + at);
        float4 x = *mine;
        if (e.w == b.w && !tile_begins(a, b)) {
            const float f = exp2f(l2 * (a.reversed ? min(b.y, b.z + SEQ_TILE) - e.z : e.z + tile_rows(e) - b.z));
            x.x = fmaf(f, before.x, x.x); x.y = fmaf(f, before.y, x.y); x.z = fmaf(f, before.z, x.z); x.w = fmaf(f, before.w, x.w);
            *mine = x;
        }
        before = x;
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
static int decay_ranges(const f3m_seqs &s, int heads) {
    int best = 1;
    float least = 0.f;
    for (int r = 1; r <= s.tiles && (r == 1 || (int64_t)heads * r <= 3 * NUM_SMS_HINT); r++) {
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
    if (p.ranges > 1) {
        static SharedMemory states;
        states.allow(decay_states<T, PARTS, NB>, bytes);
        decay_states<T, PARTS, NB><<<dim3(p.ranges - 1, p.a.heads), DS_THREADS, bytes, s>>>(p);
        F3M_LAUNCH_CHECK();
        decay_join<<<dim3((p.a.width_b * p.a.width_c / 4 + 255) / 256, p.a.heads), 256, 0, s>>>(p);
        F3M_LAUNCH_CHECK();
    }
    static SharedMemory tiles;
    tiles.allow(decay_tiles<T, PARTS, NB>, bytes);
    decay_tiles<T, PARTS, NB><<<dim3(p.ranges, p.a.heads), DK_THREADS, bytes, s>>>(p);
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
    p.mo = seq_tensor_map(Half<T>::type, a.out, a.s.tokens, a.heads, a.width_c);
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
// once, 16 bytes a thread, and that is all the time there is.
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
