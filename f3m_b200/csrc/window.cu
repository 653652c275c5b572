// Attention over a window with sinks: forward, gradients, one new token against a cache.
#include <algorithm>
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

template <typename T>
static void forward_t(const WindowArgs &a, cudaStream_t s) {
    window_rows<T, false><<<dim3(a.s.tiles * 32, a.heads), 128, 0, s>>>(a);
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
