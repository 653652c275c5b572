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
// A warp has a row, 4 columns a lane, and walks over the keys
template <typename T>
__global__ void __launch_bounds__(128) paged_rows(const __grid_constant__ PagedArgs a) {
    __shared__ uint32_t above_s[4][F3M_TREE_MAX / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, hk = h / (a.heads / a.c.kv_heads), c = 4 * lane;
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, blockIdx.x / 32)];
    const int i = e.z + 4 * (blockIdx.x % 32) + warp;
    if (i >= e.y) return;
    const int *parents = a.parents ? a.parents + e.x : nullptr;
    const int length = paged_length(a.c, e.w);
    int depth = i;
    if (parents) {
        if (lane < F3M_TREE_MAX / 32) above_s[warp][lane] = 0u;
        __syncwarp();
        depth = -1;
        for (int p = i; p >= 0; p = parent_of(parents, p), depth++)
            if (lane == 0) above_s[warp][p >> 5] |= 1u << (p & 31);
        __syncwarp();
    }
    auto read = [&](const void *p, int64_t at, float (&f)[4]) {
        uint2 v = make_uint2(0u, 0u);
        if (c + 4 <= a.c.width) v = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(p) + at + c);
        const float2 x = Half<T>::unpack(v.x), y = Half<T>::unpack(v.y);
        f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
    };
    float q[4], o[4] = {}, top = -INFINITY, sum = 0.f;
    read(a.q.data, (int64_t)(e.x + i) * a.q.token_stride + (int64_t)h * a.q.head_stride, q);
    const int64_t pos = (int64_t)length + depth, lo = max((int64_t)0, pos - a.window + 1);
    for (int64_t j = 0; j <= (int64_t)length + i; j++) {
        const int64_t m = j - length;   // a new token
        if (j < lo && j >= a.sinks && m < 0) { j = min(lo, (int64_t)length) - 1; continue; }
        if (m >= 0 && parents) {
            if (!(above_s[warp][m >> 5] >> (m & 31) & 1)) continue;
            int d = 0;
            for (int p = parent_of(parents, (int)m); p >= 0; p = parent_of(parents, p)) d++;
            if (depth - d >= a.window && length + d >= a.sinks) continue;
        } else if (j < lo && j >= a.sinks) continue;
        const int page = paged_page(a.c, e.w, j);
        if (page < 0) continue;
        float k[4], v[4];
        read(a.c.k.data, paged_at(a.c, a.c.k, page, j, hk), k);
        read(a.c.v.data, paged_at(a.c, a.c.v, page, j, hk), v);
        float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
        for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
        x *= a.scale;
        const float high = fmaxf(top, x), f = top == high ? 1.f : expf(top - high), w = expf(x - high);
        top = high;
        sum = sum * f + w;
        for (int y = 0; y < 4; y++) o[y] = o[y] * f + w * v[y];
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    if (c + 4 <= a.c.width)
        *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(a.out.data) + (int64_t)(e.x + i) * a.out.token_stride + (int64_t)h * a.out.head_stride + c) =
            make_uint2(Half<T>::pack(o[0] * inv, o[1] * inv), Half<T>::pack(o[2] * inv, o[3] * inv));
}

size_t paged_workspace(const f3m_seqs &, const f3m_cache &, int) { return 0; }

void paged_attention(int type, const PagedArgs &a, cudaStream_t s) {
    const dim3 grid(a.s.tiles * 32, a.heads);
    if (type == F3M_TYPE_BF16) paged_rows<__nv_bfloat16><<<grid, 128, 0, s>>>(a);
    else paged_rows<__half><<<grid, 128, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}

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
