// Gated recurrence by channel: forward, gradients, one new token.
#include <algorithm>
#include "seq.cuh"

namespace f3m {

// 16-byte vectors of channels as FP32
template <typename T> struct Vec {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(const void *p, int64_t i, float (&f)[8]) {
        const uint4 v = *reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p) + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 g = Half<T>::unpack(w[k]);
            f[2 * k] = g.x;
            f[2 * k + 1] = g.y;
        }
    }
    static __device__ __forceinline__ void store(void *p, int64_t i, const float (&f)[8]) {
        *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(p) + i) = make_uint4(Half<T>::pack(f[0], f[1]), Half<T>::pack(f[2], f[3]), Half<T>::pack(f[4], f[5]), Half<T>::pack(f[6], f[7]));
    }
};
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const void *p, int64_t i, float (&f)[4]) {
        const float4 v = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p) + i);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
    static __device__ __forceinline__ void store(void *p, int64_t i, const float (&f)[4]) {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + i) = make_float4(f[0], f[1], f[2], f[3]);
    }
};

// a h + x, a = exp(min(ld, 0)).  Next to 1 a's own rounding, half a step of 2^-24, would be seen in a sum over thousands of tokens: there h keeps what
// a - 1 does not take.  What is not a number stays that.
__device__ __forceinline__ float advance(float h, float ld, float x) {
    ld = ld > 0.f ? 0.f : ld;
    return ld > -0.5f ? h + fmaf(expm1f(ld), h, x) : fmaf(expf(ld), h, x);
}

template <typename T>
__global__ void __launch_bounds__(128) recurrence_walk(RecurrenceArgs a) {
    constexpr int N = Vec<T>::N;
    const int c = N * (blockIdx.x * 128 + threadIdx.x);
    if (c >= a.channels) return;
    const int4 q = reinterpret_cast<const int4 *>(a.s.table)[seq_of(a.s, blockIdx.y)];
    const int64_t at = (int64_t)blockIdx.y * a.channels + c;
    float h[N];
    for (int i = 0; i < N; i++) h[i] = a.state_in ? a.state_in[at + i] : 0.f;
    for (int64_t t = q.x; t < (int64_t)q.x + q.y; t++) {
        float x[N], ld[N];
        Vec<T>::load(a.x.data, t * a.x.token_stride + c, x);
        Vec<T>::load(a.log_decay.data, t * a.log_decay.token_stride + c, ld);
        for (int i = 0; i < N; i++) h[i] = advance(h[i], ld[i], x[i]);
        Vec<T>::store(a.out.data, t * a.out.token_stride + c, h);
    }
    if (a.state_out)
        for (int i = 0; i < N; i++) a.state_out[at + i] = h[i];
}

template <typename T>
__global__ void __launch_bounds__(128) recurrence_walk_back(RecurrenceArgs a) {
    constexpr int N = Vec<T>::N;
    const int c = N * (blockIdx.x * 128 + threadIdx.x);
    if (c >= a.channels) return;
    const int4 q = reinterpret_cast<const int4 *>(a.s.table)[seq_of(a.s, blockIdx.y)];
    const int64_t at = (int64_t)blockIdx.y * a.channels + c;
    float g[N], ld[N] = {};   // a_(t+1) G_(t+1) is taken with the next token's decay: none behind the last
    for (int i = 0; i < N; i++) g[i] = a.dstate_out ? a.dstate_out[at + i] : 0.f;
    for (int64_t t = (int64_t)q.x + q.y - 1; t >= q.x; t--) {
        float d[N], before[N], dl[N];
        Vec<T>::load(a.dout.data, t * a.dout.token_stride + c, d);
        for (int i = 0; i < N; i++) g[i] = advance(g[i], ld[i], d[i]);
        Vec<T>::store(a.dx.data, t * a.dx.token_stride + c, g);
        Vec<T>::load(a.log_decay.data, t * a.log_decay.token_stride + c, ld);
        if (t > q.x) Vec<T>::load(a.out.data, (t - 1) * a.out.token_stride + c, before);
        else
            for (int i = 0; i < N; i++) before[i] = a.state_in ? a.state_in[at + i] : 0.f;
        for (int i = 0; i < N; i++) dl[i] = ld[i] > 0.f ? 0.f : g[i] * expf(ld[i]) * before[i];
        Vec<T>::store(a.dlog_decay.data, t * a.dlog_decay.token_stride + c, dl);
    }
    if (a.dstate_in)
        for (int i = 0; i < N; i++) a.dstate_in[at + i] = advance(g[i], ld[i], 0.f);
}

// One token: a pass over the states
template <typename T>
__global__ void __launch_bounds__(256) recurrence_step_kernel(int64_t vectors, int per_row, f3m_rows x, f3m_rows log_decay, float *state, f3m_rows out) {
    constexpr int N = Vec<T>::N;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= vectors) return;
    const int64_t t = i / per_row;
    const int c = N * (int)(i % per_row);
    float f[N], ld[N], h[N];
    Vec<T>::load(x.data, t * x.token_stride + c, f);
    Vec<T>::load(log_decay.data, t * log_decay.token_stride + c, ld);
#pragma unroll
    for (int k = 0; k < N; k += 4) {
        const float4 s = *reinterpret_cast<const float4 *>(state + i * N + k);
        h[k] = advance(s.x, ld[k], f[k]);
        h[k + 1] = advance(s.y, ld[k + 1], f[k + 1]);
        h[k + 2] = advance(s.z, ld[k + 2], f[k + 2]);
        h[k + 3] = advance(s.w, ld[k + 3], f[k + 3]);
        *reinterpret_cast<float4 *>(state + i * N + k) = make_float4(h[k], h[k + 1], h[k + 2], h[k + 3]);
    }
    Vec<T>::store(out.data, t * out.token_stride + c, h);
}

size_t recurrence_workspace(const f3m_seqs &, int) { return 0; }

template <typename T>
static void walk(const RecurrenceArgs &a, bool back, cudaStream_t s) {
    F3M_REQUIRE(a.s.sequences <= 65535, F3M_ERR_UNSUPPORTED, "%d sequences in one call", a.s.sequences);
    const dim3 grid((a.channels / Vec<T>::N + 127) / 128, a.s.sequences);
    if (back) recurrence_walk_back<T><<<grid, 128, 0, s>>>(a);
    else recurrence_walk<T><<<grid, 128, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}
static void walk_type(int type, const RecurrenceArgs &a, bool back, cudaStream_t s) {
    if (type == F3M_TYPE_BF16) walk<__nv_bfloat16>(a, back, s);
    else if (type == F3M_TYPE_F16) walk<__half>(a, back, s);
    else walk<float>(a, back, s);
}
void recurrence_forward(int type, const RecurrenceArgs &a, cudaStream_t s) { walk_type(type, a, false, s); }
void recurrence_backward(int type, const RecurrenceArgs &a, cudaStream_t s) { walk_type(type, a, true, s); }

template <typename T>
static void step_t(int n, int channels, const f3m_rows &x, const f3m_rows &log_decay, float *state, const f3m_rows &out, cudaStream_t s) {
    const int per_row = channels / Vec<T>::N;
    const int64_t vectors = (int64_t)n * per_row, blocks = (vectors + 255) / 256;
    F3M_REQUIRE(blocks <= 0x7fffffff, F3M_ERR_OVERFLOW, "%d sequences of %d channels do not fit in 31 bits", n, channels);
    recurrence_step_kernel<T><<<(unsigned)blocks, 256, 0, s>>>(vectors, per_row, x, log_decay, state, out);
    F3M_LAUNCH_CHECK();
}
void recurrence_step(int type, int n, int channels, const f3m_rows &x, const f3m_rows &log_decay, float *state, const f3m_rows &out, cudaStream_t s) {
    if (type == F3M_TYPE_BF16) step_t<__nv_bfloat16>(n, channels, x, log_decay, state, out, s);
    else if (type == F3M_TYPE_F16) step_t<__half>(n, channels, x, log_decay, state, out, s);
    else step_t<float>(n, channels, x, log_decay, state, out, s);
}

}  // namespace f3m
