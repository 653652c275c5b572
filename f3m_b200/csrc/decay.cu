// Linear attention with a decay for each head: the recurrence over packed sequences, and one new token.
#include "seq.cuh"

namespace f3m {

// A CTA per (sequence, head) walks the tokens; thread c holds column c of the state.
template <typename T>
__global__ void __launch_bounds__(128) decay_walk(DecayArgs a) {
    __shared__ float as[F3M_MAX_WIDTH], bs[F3M_MAX_WIDTH];
    const int4 e = reinterpret_cast<const int4 *>(a.s.table)[seq_of(a.s, blockIdx.x)];
    const int h = blockIdx.y, c = threadIdx.x, wb = a.width_b, wc = a.width_c;
    const float decay = exp2f(log2_decay(a.log_decay[h]));
    const int64_t base = ((int64_t)blockIdx.x * a.heads + h) * wb * wc;
    float S[F3M_MAX_WIDTH];
#pragma unroll
    for (int d = 0; d < F3M_MAX_WIDTH; d++) S[d] = a.state_in && c < wc && d < wb ? a.state_in[base + (a.transposed ? (int64_t)c * wb + d : (int64_t)d * wc + c)] : 0.f;
    for (int n = 0; n < e.y; n++) {
        const int64_t t = e.x + (a.reversed ? e.y - 1 - n : n);
        __syncthreads();
        if (c < wb) {
            as[c] = (float)(reinterpret_cast<const T *>(a.a.data)[t * a.a.token_stride + h * a.a.head_stride + c]);
            bs[c] = (float)(reinterpret_cast<const T *>(a.b.data)[t * a.b.token_stride + h * a.b.head_stride + c]);
        }
        __syncthreads();
        const float cv = c < wc ? a.upd * (float)(reinterpret_cast<const T *>(a.c.data)[t * a.c.token_stride + h * a.c.head_stride + c]) : 0.f;
        float o = 0.f;
#pragma unroll
        for (int d = 0; d < F3M_MAX_WIDTH; d++)
            if (d < wb) {
                S[d] = (a.reversed && n == 0 ? S[d] : decay * S[d]) + bs[d] * cv;
                o = fmaf(as[d], S[d], o);
            }
        if (c < wc) reinterpret_cast<T *>(a.out.data)[t * a.out.token_stride + h * a.out.head_stride + c] = (T)(a.use * o);
    }
    if (a.state_out && c < wc)
#pragma unroll
        for (int d = 0; d < F3M_MAX_WIDTH; d++)
            if (d < wb) a.state_out[base + (a.transposed ? (int64_t)c * wb + d : (int64_t)d * wc + c)] = a.reversed && e.y ? decay * S[d] : S[d];
}

size_t decay_workspace(const f3m_seqs &, int, int, int) { return 0; }
void decay_product(int type, const DecayArgs &a, cudaStream_t s) {
    if (type == F3M_TYPE_BF16) decay_walk<__nv_bfloat16><<<dim3(a.s.sequences, a.heads), 128, 0, s>>>(a);
    else decay_walk<__half><<<dim3(a.s.sequences, a.heads), 128, 0, s>>>(a);
    F3M_LAUNCH_CHECK();
}

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
