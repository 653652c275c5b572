// What the kernel products over sequences share: arguments, 16-bit types, the table of tiles.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"
#include "packed.cuh"
#include "tc.cuh"

namespace f3m {

constexpr int SEQ_TILE = F3M_SEQ_TILE;

// The table of a packed batch, as int4: three orders of the tiles {first row of the sequence, its length, first token of the tile, sequence}
// -- by place, by the tokens before the tile (the rows of late tiles see the most keys) and by the tokens from it on (the keys of early
// tiles are seen most), the heaviest first in both -- behind them the sequences {first row, length, first tile, tiles}, and behind those every other
// tile of each sequence, from its first on, in the second order.
__host__ __device__ __forceinline__ size_t seq_by_place(const f3m_seqs &, int i) { return (size_t)i; }
__host__ __device__ __forceinline__ size_t seq_by_past(const f3m_seqs &s, int i) { return (size_t)s.tiles + i; }
__host__ __device__ __forceinline__ size_t seq_by_future(const f3m_seqs &s, int i) { return 2 * (size_t)s.tiles + i; }
__host__ __device__ __forceinline__ size_t seq_of(const f3m_seqs &s, int i) { return 3 * (size_t)s.tiles + i; }

__host__ __device__ __forceinline__ size_t seq_pair_by_past(const f3m_seqs &s, int i) { return 3 * (size_t)s.tiles + s.sequences + i; }

template <typename T> struct Half;
template <> struct Half<__nv_bfloat16> {
    static constexpr int type = F3M_TYPE_BF16;
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {   // round to nearest even
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct Half<__half> {
    static constexpr int type = F3M_TYPE_F16;
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        const __half2 h = *reinterpret_cast<const __half2 *>(&v);
        return __half22float2(h);
    }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};

// 2^x of two numbers on the FMA pipe, for x up to 126: x = n + f with |f| <= 1/2, a polynomial of degree 4 for 2^f (least maximum of the relative
// error on that interval, 2.6e-6, by Lawson's iteration), times 2^n.  Below -125 it stays at 2^-125.  Takes part of the exponentials
// off the special-function unit, which gives 16 a clock and SM, and nothing it is used for is kept to more than 16 bits but sums of many of them.
// KEEP_NAN: 2^n is multiplied in, and what is not a number stays that.  Otherwise n is added to the exponent's bits, an instruction less for two, and what is
// not a number becomes FP32's largest one, infinite as an operand: the sum that it goes into has to be looked at.  (In window_tiles the product takes 1.4 %.)
template <bool KEEP_NAN>
__device__ __forceinline__ void exp2_poly(f32x2 x, float &lo, float &hi) {
    float a, b;
    unpack2(x, a, b);
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-125.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-125.f));
    x = pack2(a, b);
    const f32x2 magic = pack2(12582912.f, 12582912.f), t = add2(x, magic), n = add2(t, pack2(-12582912.f, -12582912.f)), f = fma2(n, pack2(-1.f, -1.f), x);
    f32x2 y = fma2(pack2(0.009570102f, 0.009570102f), f, pack2(0.055917863f, 0.055917863f));
    y = fma2(y, f, pack2(0.24024744f, 0.24024744f));
    y = fma2(y, f, pack2(0.69312179f, 0.69312179f));
    y = fma2(y, f, pack2(0.99999928f, 0.99999928f));
    float tl, th;
    unpack2(t, tl, th);
    if (KEEP_NAN) {
        unpack2(mul2(y, pack2(__uint_as_float((__float_as_uint(tl) << 23) + 0x3f800000u), __uint_as_float((__float_as_uint(th) << 23) + 0x3f800000u))), lo, hi);
    } else {
        unpack2(y, a, b);
        lo = __uint_as_float(__float_as_uint(a) + (__float_as_uint(tl) << 23));
        hi = __uint_as_float(__float_as_uint(b) + (__float_as_uint(th) << 23));
    }
}

struct WindowArgs {
    f3m_seqs s;
    int heads, kv_heads, width, window, sinks;
    float scale;
    f3m_rows q, k, v, out;
    float *lse;
    f3m_rows dout, dq, dk, dv;   // gradients only
    float *delta;                // workspace: 2 x (heads, tokens), (sequences, kv_heads, 2), and the parts' sums
};
void window_forward(int type, const WindowArgs &a, cudaStream_t s);
void window_backward(int type, const WindowArgs &a, cudaStream_t s);
size_t window_grad_workspace(const f3m_seqs &s, int heads, int kv_heads, int width, int window, int sinks);

struct StepArgs {
    int n, heads, kv_heads, width, window, sinks;
    int64_t capacity;
    float scale;
    f3m_rows q, k, v, out;
    int64_t k_seq, v_seq;
    const int *lengths;
    int parts;      // splits of the keys
    float *part;    // their sums
};
int window_step_parts(int n, int heads, int kv_heads, int64_t capacity, int window, int sinks);
size_t window_step_part_floats(int n, int heads, int width, int parts);
void window_step(int type, const StepArgs &a, cudaStream_t s);

// out_i = use * sum_(j before or at i) decay^|i-j| upd (a_i.b_j) c_j + use * decay^(steps to i) a_i S, S (width of b, width of c).
// `reversed`: sequences run from their last token to their first; the state that enters does so undecayed, the one that
// leaves has been decayed once more (the adjoint of the recurrence).  `transposed`: states lie in memory as (width of c, width of b).
struct DecayArgs {
    f3m_seqs s;
    int heads, width_b, width_c;
    const float *log_decay;
    float use, upd;
    bool reversed, transposed;
    bool joined;   // ws holds the states between ranges already, as the same product with b and c exchanged left them
    f3m_rows a, b, c, out;
    const float *state_in;
    float *state_out;
    void *ws;
};
size_t decay_workspace(const f3m_seqs &s, int heads, int width_b, int width_c);
void decay_product(int type, const DecayArgs &a, cudaStream_t s);
void decay_step(int type, int n, int heads, int width_k, int width_v, const float *log_decay, float scale, const f3m_rows &q, const f3m_rows &k,
                const f3m_rows &v, float *state, const f3m_rows &out, cudaStream_t s);

// A tensor map of (tokens, heads, width) rows whose boxes are 64 columns x 1 head x 128 tokens, swizzled
CUtensorMap seq_tensor_map(int type, const f3m_rows &r, int64_t tokens, int heads, int width);
// The word in mapped host memory where a kernel notes that a wait of its ran out; the next call reports it
int *seq_error_word();
void seq_check_error();

// A kernel's leave to use more than 48 KB of shared memory, asked for once on each device
class SharedMemory {
    std::atomic<unsigned long long> devices{0};   // the first 64; others ask each time
public:
    template <typename K>
    void allow(K kernel, int bytes) {
        int d = 0;
        F3M_CUDA(cudaGetDevice(&d));
        if (d < 64 && devices.load(std::memory_order_relaxed) >> d & 1) return;
        F3M_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (d < 64) devices.fetch_or(1ull << d, std::memory_order_relaxed);
    }
};

// Waits of a kernel's roles on one another.  None is longer than about two seconds (a try lasts two microseconds at most): what expires raises
// `gave_up`, after which every wait of the block returns at once and the block runs to its end on whatever it finds, inside its buffers. 
constexpr uint32_t WAIT_TRIES = 1000000;
struct Waits {
    volatile int *gave_up;
    int *err;
    __device__ __forceinline__ void operator()(uint32_t bar, uint32_t parity) const {
        uint32_t tries = 0;
        while (!tc::mbar_try_wait_ns(bar, parity, 2000))
            if (*gave_up || ++tries > WAIT_TRIES) {
                *gave_up = 1;
                *(volatile int *)err = 1;
                return;
            }
    }
    // also when the block has given up: copies in flight are waited for before it ends
    __device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) const {
        for (uint32_t tries = 0; tries < WAIT_TRIES && !tc::mbar_try_wait_ns(bar, parity, 2000); tries++) {}
    }
    // by the warp that issues the block's products, behind the last of them: where the block has given up, nobody else may have waited for those in flight, and the
    // tensor memory that they write is about to be another block's
    __device__ __forceinline__ void drain_products(uint32_t bar) const {
        if (__any_sync(0xffffffffu, *gave_up) && tc::elect()) {
            tc::mma_commit(bar);
            drain(bar, 0);
        }
    }
};

__device__ __forceinline__ void sts16(uint32_t at, const uint32_t (&w)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}
// Chunks [c0, c1) of row j of a tile become zero: tokens of the next sequence meet no weight, not even a weight of zero
__device__ __forceinline__ void clear_row(uint32_t tile, int j, int c0, int c1) {
    const uint32_t zero[4] = {0u, 0u, 0u, 0u};
#pragma unroll 1
    for (int i = c0; i < c1; i++) sts16(tile + (i >> 3) * SEQ_TILE * 128 + tc::swz(j, i & 7), zero);
}

// 32 columns of a row, 16 bits each, to memory; `wide`: the row starts on 32 bytes.  Rows go straight from registers: a thread writes whole sectors.
// (Staged in shared memory and sent as bulk copies, a tile's rows held their stage for another 1600 to 10000 clocks.)
__device__ __forceinline__ void store_row32(uint16_t *row, const uint32_t (&w)[16], int c0, int width, bool wide) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint16_t *at = row + c0 + 16 * h;
        if (wide && c0 + 16 * h + 16 <= width)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[8 * h]), "r"(w[8 * h + 1]), "r"(w[8 * h + 2]), "r"(w[8 * h + 3]),
                         "r"(w[8 * h + 4]), "r"(w[8 * h + 5]), "r"(w[8 * h + 6]), "r"(w[8 * h + 7])
                         : "memory");
        else {
            if (c0 + 16 * h < width) *reinterpret_cast<uint4 *>(at) = make_uint4(w[8 * h], w[8 * h + 1], w[8 * h + 2], w[8 * h + 3]);
            if (c0 + 16 * h + 8 < width) *reinterpret_cast<uint4 *>(at + 8) = make_uint4(w[8 * h + 4], w[8 * h + 5], w[8 * h + 6], w[8 * h + 7]);
        }
    }
}
__host__ __device__ __forceinline__ bool rows_wide(const f3m_rows &r) { return (uintptr_t)r.data % 32 == 0 && r.token_stride % 16 == 0 && r.head_stride % 16 == 0; }

// Rows 0 .. m of a swizzled tile in shared memory, columns from col0 on, to tokens token .. token + m, by THREADS threads (t) that have each written rows of it;
// on return thread 0 knows that the tile has been read.  A whole tile leaves as bulk copies; one that ends inside would write over the
// next sequence's rows, so its rows are written one by one.
template <int THREADS>
__device__ __forceinline__ void store_rows(const CUtensorMap &map, const f3m_rows &out, uint32_t tile, int head, int token, int m, int col0, int blocks,
                                           int width, int t, int barrier) {
    if (m == SEQ_TILE) {
        tc::fence_async_smem();
        tc::bar_sync(barrier, THREADS);
        if (t == 0) {
#pragma unroll 1
            for (int k = 0; k < blocks; k++) tc::tma_store_rows(&map, tile + k * SEQ_TILE * 128, col0 + 64 * k, head, token);
            tc::tma_store_commit();
            tc::tma_store_wait_read();
        }
    } else {
        tc::bar_sync(barrier, THREADS);
#pragma unroll 1
        for (int i = t; i < m * 8 * blocks; i += THREADS) {   // 16-byte chunks; consecutive threads along a row
            const int r = i / (8 * blocks), c = i % (8 * blocks);
            uint32_t v[4];
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(tile + (c >> 3) * SEQ_TILE * 128 + tc::swz(r, c & 7)) : "memory");
            if (col0 + 8 * c < width)
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(out.data) + (int64_t)(token + r) * out.token_stride + (int64_t)head * out.head_stride + col0 + 8 * c) = make_uint4(v[0], v[1], v[2], v[3]);
        }
        tc::bar_sync(barrier, THREADS);
    }
}

// log2 of a head's decay: at most 0; -256 makes every power but the zeroth 0 in FP32 and keeps 0 * log a number.  What is not a number stays that.
__device__ __forceinline__ float log2_decay(float log_decay) {
    const float x = log_decay * 1.4426950408889634f;
    return x > 0.f ? 0.f : x < -256.f ? -256.f : x;
}

}  // namespace f3m
