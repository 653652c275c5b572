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

// ---- whole sequences --------------------------------------------------------------------------------------------------------
// A unit is a tile of 128 tokens by 128 bytes of channels, a lane two channels.  Its tokens are cut into runs, one for 32 or 16 lanes each; a run is the map h -> A h + B, with
// A from the sum of its log decays, and so is the tile.  What enters a tile is found by looking back over the tiles before it, of which each tells its map as soon as it
// has it, and what leaves it as soon as it knows what entered: the nearest such state goes through the maps in between, always one after the other, so that a call's bits
// do not depend on how far that was.  Then every run is walked again, from what enters it.  Each array is read and written once.
//
// Gradients are the same from the end, on what flows back between tokens, c_t = a_t G_t: G_t = dout_t + c_(t+1), dx_t = G_t, dlog_decay_t = c_t h_(t-1).
//
// Blocks take units from a counter, tiles in order, so that what a tile waits for is always taken by a running block; a ninth warp takes the next one, starts its
// copies, and looks back.
constexpr int GR_WARPS = 8, GR_THREADS = 32 * (GR_WARPS + 1), GR_TILE = SEQ_TILE * 128;   // bytes of an array's tile
template <bool BACK> constexpr int GR_STAGES = BACK ? 2 : 3;
enum { GR_NOTHING = 0, GR_MAP = 1, GR_STATE = 2 };   // what a tile has told

struct RecurrenceKernel {
    RecurrenceArgs a;
    CUtensorMap m[3];   // x, log_decay; or dout, log_decay, out
    int groups;         // of channels
    int units;
    bool counted;       // tiles look back: units come from the counter
    int *told;          // the counter, and from word 4 on by unit
    float4 *maps;       // by unit and lane: multipliers of its two channels, added
    float2 *states;     // what left
    int *err;
};

// Multipliers: a or, where it is above exp(-1/4), a - 1, which is told by its sign (-0 for a decay of 1).  A decay next to 1 that is rounded to FP32 would leave a sum
// over thousands of tokens 1e-5 off; a - 1 keeps its bits, as ld (1 + ld / 2 + ld^2 / 6 + ..) to the sixth power, 5e-8 off at most.
__device__ __forceinline__ f32x2 multiplier(f32x2 ld) {
    f32x2 y = fma2(ld, pack2(1.f / 720, 1.f / 720), pack2(1.f / 120, 1.f / 120));
    y = fma2(y, ld, pack2(1.f / 24, 1.f / 24));
    y = fma2(y, ld, pack2(1.f / 6, 1.f / 6));
    y = fma2(y, ld, pack2(0.5f, 0.5f));
    y = mul2(fma2(y, ld, pack2(1.f, 1.f)), ld);
    float near[2], far[2], l[2];
    unpack2(y, near[0], near[1]);
    unpack2(ld, l[0], l[1]);
    unpack2(mul2(ld, pack2(1.4426950408889634f, 1.4426950408889634f)), far[0], far[1]);
    return pack2(l[0] > -0.25f ? near[0] : ex2_approx(far[0]), l[1] > -0.25f ? near[1] : ex2_approx(far[1]));   // what is not a number stays that
}
// a h + x
__device__ __forceinline__ f32x2 through(f32x2 h, f32x2 m, f32x2 x) {
    float hl, hh, ml, mh;
    unpack2(h, hl, hh);
    unpack2(m, ml, mh);
    const f32x2 kept = pack2(__int_as_float(__float_as_int(hl) & __float_as_int(ml) >> 31), __int_as_float(__float_as_int(hh) & __float_as_int(mh) >> 31));
    return add2(fma2(m, h, x), kept);
}
__device__ __forceinline__ f32x2 held(f32x2 ld) {   // at most -0
    float l, h;
    unpack2(ld, l, h);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(l) : "f"(-0.f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(h) : "f"(-0.f));
    return pack2(l, h);
}

// Two channels as they lie in memory
template <typename T> struct Two {
    typedef uint32_t Raw;
    static __device__ __forceinline__ f32x2 open(Raw v) { const float2 f = Half<T>::unpack(v); return pack2(f.x, f.y); }
    static __device__ __forceinline__ Raw close(f32x2 v) { float l, h; unpack2(v, l, h); return Half<T>::pack(l, h); }
};
template <> struct Two<float> {
    typedef unsigned long long Raw;
    static __device__ __forceinline__ f32x2 open(Raw v) { return v; }
    static __device__ __forceinline__ Raw close(f32x2 v) { return v; }
};

template <typename T, bool BACK>
__global__ void __launch_bounds__(GR_THREADS, 2) recurrence_tiles(const __grid_constant__ RecurrenceKernel p) {
    typedef typename Two<T>::Raw Raw;
    constexpr int ARRAYS = BACK ? 3 : 2, STAGES = GR_STAGES<BACK>, LANES = 128 / sizeof(Raw), RUNS = GR_WARPS * 32 / LANES, RUN = SEQ_TILE / RUNS, CHANNELS = 2 * LANES;
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[STAGES];
    __shared__ __align__(16) float4 runs_s[RUNS][LANES];   // maps of the runs: sums of log decays, added
    __shared__ f32x2 enter_s[RUNS][LANES];
    __shared__ int unit_s[STAGES], gave_up_s;
    const RecurrenceArgs &a = p.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned char *base = raw + (-tc::smem_u32(raw) & 127);
    const uint32_t smem = tc::smem_u32(base), b_full = tc::smem_u32(&bars[0]);
    const f32x2 none = pack2(-0.f, -0.f);   // the log of no decay, summed
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; i++) tc::mbar_init(b_full + 8 * i, 1);
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    __syncthreads();
    const Waits wait{&gave_up_s, p.err};
    auto entry = [&](int u) {   // {first row, length, first token, sequence}
        const int i = u / p.groups;
        return reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, BACK ? a.s.tiles - 1 - i : i)];
    };
    int taken = (int)blockIdx.x - (int)gridDim.x, copies = 0;   // of the ninth warp's first lane
    auto take = [&](int stage) {   // the next unit, and its copies
        taken = p.counted ? atomicAdd(p.told, 1) : taken + (int)gridDim.x;
        unit_s[stage] = min(taken, p.units);
        if (taken >= p.units) return;
        const int4 e = entry(taken);
        tc::mbar_expect_tx(b_full + 8 * stage, ARRAYS * GR_TILE);
        for (int i = 0; i < ARRAYS; i++)   // of the outputs the tokens before
            tc::tma_rows(smem + (ARRAYS * stage + i) * GR_TILE, &p.m[i], taken % p.groups * CHANNELS, 0, e.x + e.z - (i == 2), b_full + 8 * stage);
        copies++;
    };
    if (threadIdx.x == 32 * GR_WARPS)
        for (int i = 0; i < STAGES - 1; i++) take(i);
    for (int n = 0;; n++) {
        __syncthreads();   // the unit is known, and all have done with the one before
        const int stage = n % STAGES, u = unit_s[stage];
        if (u >= p.units) break;
        const int4 e = entry(u);
        const int g = u % p.groups, count = min(SEQ_TILE, e.y - e.z);
        if (warp == GR_WARPS) {
            if (lane == 0) take((n + STAGES - 1) % STAGES);
            __syncwarp();
            const int before = BACK ? (e.y - 1) / SEQ_TILE - e.z / SEQ_TILE : e.z / SEQ_TILE;   // tiles before this one
            const bool last = BACK ? e.z == 0 : e.z + SEQ_TILE >= e.y;
            const int l = lane % LANES, c = g * CHANNELS + 2 * l;
            const float *in = BACK ? a.dstate_out : a.state_in;   // what enters the sequence, and leaves it
            float *out = BACK ? a.dstate_in : a.state_out;
            const bool mine = lane < LANES && c < a.channels;
            f32x2 h = 0;
            if (before == 0 && in && c < a.channels) h = *reinterpret_cast<const f32x2 *>(in + (int64_t)e.w * a.channels + c);
            auto run = [&](int i, f32x2 &log, f32x2 &added) {
                const float4 r = runs_s[BACK ? RUNS - 1 - i : i][l];
                log = pack2(r.x, r.y);
                added = pack2(r.z, r.w);
            };
            __syncthreads();   // the runs' maps are there
            f32x2 leaves = 0;   // told to the tiles behind: through the tile's own map, as those do who look over it
            if (before) {
                int *told = p.told + 4 + u;
                f32x2 logs = none, sum = 0;
                if (!last) {
#pragma unroll 4
                    for (int i = 0; i < RUNS; i++) {
                        f32x2 log, added;
                        run(i, log, added);
                        logs = add2(logs, log);
                        sum = through(sum, multiplier(log), added);
                    }
                    float4 map;
                    unpack2(multiplier(logs), map.x, map.y);
                    unpack2(sum, map.z, map.w);
                    if (lane < LANES) __stcg(p.maps + (int64_t)u * LANES + l, map);
                    __threadfence();
                    __syncwarp();
                    if (lane == 0) *(volatile int *)told = GR_MAP;
                }
                // the nearest tile that has told what left it, with maps told by all in between
                int near = 0;
                for (uint32_t tries = 0;;) {
                    const int what = lane < before ? *(volatile int *)(told - (int64_t)p.groups * (1 + lane)) : GR_NOTHING;
                    const uint32_t has = __ballot_sync(0xffffffffu, what == GR_STATE), nothing = __ballot_sync(0xffffffffu, what == GR_NOTHING);
                    near = __ffs(has) - 1;
                    if (has && (nothing & ((1u << near) - 1)) == 0) break;
                    if (__any_sync(0xffffffffu, gave_up_s) || ++tries > 2 * WAIT_TRIES) {   // a try takes a microsecond, about
                        if (lane == 0) {
                            gave_up_s = 1;
                            *(volatile int *)p.err = 1;
                        }
                        near = 0;
                        break;
                    }
                    __nanosleep(50);
                }
                __threadfence();
                const float2 s = __ldcg(p.states + (int64_t)(u - p.groups * (1 + near)) * LANES + l);
                h = pack2(s.x, s.y);
#pragma unroll 4
                for (int i = near - 1; i >= 0; i--) {
                    const float4 map = __ldcg(p.maps + (int64_t)(u - p.groups * (1 + i)) * LANES + l);
                    h = through(h, pack2(map.x, map.y), pack2(map.z, map.w));
                }
                leaves = through(h, multiplier(logs), sum);
            }
#pragma unroll 4
            for (int i = 0; i < RUNS; i++) {
                f32x2 log, added;
                run(i, log, added);
                if (lane < LANES) enter_s[BACK ? RUNS - 1 - i : i][l] = h;
                h = through(h, multiplier(log), added);
            }
            __syncthreads();   // what enters the runs is there
            if (last) {
                if (out && mine) *reinterpret_cast<f32x2 *>(out + (int64_t)e.w * a.channels + c) = h;
            } else {
                float2 s;
                unpack2(before ? leaves : h, s.x, s.y);
                if (lane < LANES) __stcg(p.states + (int64_t)u * LANES + l, s);
                __threadfence();
                __syncwarp();
                if (lane == 0) *(volatile int *)(p.told + 4 + u) = GR_STATE;
            }
        } else {
            const int run = warp * (32 / LANES) + lane / LANES, l = lane % LANES, r0 = run * RUN, c = g * CHANNELS + 2 * l;
            const unsigned char *tile = base + ARRAYS * stage * GR_TILE + r0 * 128 + l * sizeof(Raw);
            auto raw_of = [&](int array, int i) { return *reinterpret_cast<const Raw *>(tile + array * GR_TILE + i * 128); };
            f32x2 m[RUN], logs = none, sum = 0;
            Raw x[RUN];   // x, or dout
            wait(b_full + 8 * stage, (n / STAGES) & 1);
#pragma unroll
            for (int k = 0; k < RUN; k++) {
                const int i = BACK ? RUN - 1 - k : k;
                x[i] = raw_of(0, i);
                f32x2 ld = held(Two<T>::open(raw_of(1, i)));
                if (r0 + i >= count) { x[i] = 0; ld = none; }   // behind the sequence
                m[i] = multiplier(ld);
                logs = add2(logs, ld);
                sum = BACK ? through(add2(sum, Two<T>::open(x[i])), m[i], 0) : through(sum, m[i], Two<T>::open(x[i]));
            }
            float4 map;
            unpack2(logs, map.x, map.y);
            unpack2(sum, map.z, map.w);
            runs_s[run][l] = map;
            __syncthreads();   // the runs' maps are there
            __syncthreads();   // what enters the runs is there
            f32x2 h = enter_s[run][l];
            const int64_t t0 = (int64_t)e.x + e.z + r0;
            const int rows = c < a.channels ? count - r0 : 0;   // of this run's
            T *y = reinterpret_cast<T *>(BACK ? a.dx.data : a.out.data) + t0 * (BACK ? a.dx.token_stride : a.out.token_stride) + c;
            T *z = BACK ? reinterpret_cast<T *>(a.dlog_decay.data) + t0 * a.dlog_decay.token_stride + c : nullptr;
#pragma unroll
            for (int k = 0; k < RUN; k++) {
                const int i = BACK ? RUN - 1 - k : k;
                if constexpr (!BACK) {
                    h = through(h, m[i], Two<T>::open(x[i]));
                    if (i < rows) *reinterpret_cast<Raw *>(y + i * a.out.token_stride) = Two<T>::close(h);
                } else {
                    const f32x2 d = add2(h, Two<T>::open(x[i]));
                    h = through(d, m[i], 0);
                    if (i >= rows) continue;
                    *reinterpret_cast<Raw *>(y + i * a.dx.token_stride) = Two<T>::close(d);
                    f32x2 past = Two<T>::open(raw_of(2, i));
                    if (e.z + r0 + i == 0) past = a.state_in ? *reinterpret_cast<const f32x2 *>(a.state_in + (int64_t)e.w * a.channels + c) : 0;
                    float ll, lh, dl, dh;
                    unpack2(Two<T>::open(raw_of(1, i)), ll, lh);
                    unpack2(mul2(h, past), dl, dh);
                    *reinterpret_cast<Raw *>(z + i * a.dlog_decay.token_stride) = Two<T>::close(pack2(ll > 0.f ? 0.f : dl, lh > 0.f ? 0.f : dh));
                }
            }
        }
    }
    if (threadIdx.x == 32 * GR_WARPS && copies)   // copies that nobody waited for, where the block gave up
        for (int i = max(0, copies - STAGES); i < copies; i++) wait.drain(b_full + 8 * (i % STAGES), (i / STAGES) & 1);
}

// Sequences without tokens
__global__ void __launch_bounds__(256) recurrence_empty(f3m_seqs s, int channels, const float *in, float *out) {
    const int64_t at = (int64_t)blockIdx.x * channels;
    if (reinterpret_cast<const int4 *>(s.table)[seq_of(s, blockIdx.x)].y) return;
    for (int c = threadIdx.x; c < channels; c += 256) out[at + c] = in ? in[at + c] : 0.f;
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

// the counter and what the tiles have told, maps, states; more than enough for any type
static size_t told_bytes(const f3m_seqs &s, int channels) { return 16 + ((size_t)s.tiles * ((channels + 31) / 32) * 4 + 15) / 16 * 16; }
static size_t lane_places(const f3m_seqs &s, int channels) { return (size_t)s.tiles * ((channels + 63) / 64) * 32; }
size_t recurrence_workspace(const f3m_seqs &s, int channels) {
    return s.longest > SEQ_TILE ? told_bytes(s, channels) + lane_places(s, channels) * (sizeof(float4) + sizeof(float2)) : 0;
}

template <typename T, bool BACK>
static void recurrence_t(int type, const RecurrenceArgs &a, cudaStream_t s) {
    if (a.s.empty) {
        const float *in = BACK ? a.dstate_out : a.state_in;
        float *out = BACK ? a.dstate_in : a.state_out;
        if (out) {
            recurrence_empty<<<a.s.sequences, 256, 0, s>>>(a.s, a.channels, in, out);
            F3M_LAUNCH_CHECK();
        }
    }
    if (a.s.tokens == 0) return;
    RecurrenceKernel p;
    p.a = a;
    constexpr int channels = 128 / sizeof(T);
    const int arrays = BACK ? 3 : 2;
    p.groups = (a.channels + channels - 1) / channels;
    F3M_REQUIRE((int64_t)a.s.tiles * p.groups <= 0x7fff0000, F3M_ERR_OVERFLOW, "%d tiles of %d channels do not fit in 31 bits", a.s.tiles, a.channels);
    p.units = a.s.tiles * p.groups;
    p.counted = a.s.longest > SEQ_TILE;
    p.told = reinterpret_cast<int *>(a.ws);
    p.maps = reinterpret_cast<float4 *>(reinterpret_cast<char *>(a.ws) + told_bytes(a.s, a.channels));
    p.states = reinterpret_cast<float2 *>(p.maps + lane_places(a.s, a.channels));
    p.err = seq_error_word();
    p.m[0] = channel_tensor_map(type, BACK ? a.dout : a.x, a.s.tokens, a.channels);
    p.m[1] = channel_tensor_map(type, a.log_decay, a.s.tokens, a.channels);
    if (BACK) p.m[2] = channel_tensor_map(type, a.out, a.s.tokens, a.channels);
    if (p.counted) F3M_CUDA(cudaMemsetAsync(p.told, 0, 16 + 4 * (size_t)p.units, s));
    const int bytes = GR_STAGES<BACK> * arrays * GR_TILE + 128;
    static SharedMemory allowed;
    allowed.allow(recurrence_tiles<T, BACK>, bytes);
    recurrence_tiles<T, BACK><<<std::min(p.units, 2 * NUM_SMS_HINT), GR_THREADS, bytes, s>>>(p);
    F3M_LAUNCH_CHECK();
}
template <bool BACK>
static void recurrence_type(int type, const RecurrenceArgs &a, cudaStream_t s) {
    if (type == F3M_TYPE_BF16) recurrence_t<__nv_bfloat16, BACK>(type, a, s);
    else if (type == F3M_TYPE_F16) recurrence_t<__half, BACK>(type, a, s);
    else recurrence_t<float, BACK>(type, a, s);
}
void recurrence_forward(int type, const RecurrenceArgs &a, cudaStream_t s) { recurrence_type<false>(type, a, s); }
void recurrence_backward(int type, const RecurrenceArgs &a, cudaStream_t s) { recurrence_type<true>(type, a, s); }

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
