// Gated recurrence by channel: forward, gradients, one new token.
#include <algorithm>
#include <type_traits>
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
// a - 1 does not take.  What is not a number stays that.  An infinite h has nothing to keep, and a - 1 would turn its sign: it is a's multiple, infinite where a is above 0 as the
// kernels of whole sequences take it (decay_of).
__device__ __forceinline__ float advance(float h, float ld, float x) {
    ld = ld > 0.f ? 0.f : ld;
    if (isinf(h)) return fmaf(ex2_approx(1.4426950408889634f * ld), h, x);
    return ld > -0.5f ? h + fmaf(expm1f(ld), h, x) : fmaf(expf(ld), h, x);
}

// ---- whole sequences --------------------------------------------------------------------------------------------------------
// A scan in one pass with look-back (D. Merrill and M. Garland, 2016).  A unit is a tile of 128 tokens by 128 bytes of channels, a lane two channels.  Its tokens are cut into runs, one for 32 or 16 lanes each; a run is the map h -> A h + B, with
// A from the sum of its log decays, and so is the tile.  What enters a tile is found by looking back over the tiles before it, of which each tells its map as soon as it
// has it, and what leaves it as soon as it knows what entered: the nearest such state goes through the maps in between, always one after the other, so that a call's bits
// do not depend on how far that was.  Then every run is walked again, from what enters it.  Each array is read and written once.
//
// Maps and states are told in words of 8 bytes that are all ones before, which no number here is: a word is there when it is another, and needs no flag and no fence.
//
// Gradients are the same from the end, on what flows back between tokens, c_t = a_t G_t: G_t = dout_t + c_(t+1), dx_t = G_t, dlog_decay_t = c_t h_(t-1).
//
// What bounds it: the steps of a unit, which wait for one another (copies, first walk, fold, looking back, second walk with its stores), and three units on an SM (two of gradients), which do not fill them.
// 65536 tokens, 2048 channels, bf16: 217 us, 3.7 TB/s (fp32 354 us, 4.5; gradients 319 and 551 us, 4.2 and 4.9), 5.9 us a unit, or 11600 clocks at 1965 MHz; 1200 go to each walk, and more than
// half to looking back, as the tiles before run at the same time.  64 sequences of 128 tokens, 4096 channels, where nothing looks back: 43 us, 4.8 TB/s.
//
// Blocks take units from a counter, tiles in order, so that what a tile waits for is always taken by a running block; a ninth warp takes the next one, starts its
// copies, and looks back.
constexpr int GR_WARPS = 8, GR_THREADS = 32 * (GR_WARPS + 1), GR_TILE = SEQ_TILE * 128, GR_STAGES = 2;   // bytes of an array's tile
constexpr unsigned long long GR_NOTHING = ~0ull;
constexpr int GR_MAPS = 4;   // words of so many tiles on their way at a time: 218 us, one by one 238 (65536 tokens, 2048 channels); eight spill

struct RecurrenceKernel {
    RecurrenceArgs a;
    CUtensorMap m[3];   // x, log_decay; or dout, log_decay, out
    int groups;         // of channels
    int units;
    bool counted;       // tiles look back: units come from the counter
    unsigned *counter;  // all ones before the first
    unsigned long long *told;   // by unit and lane: multipliers, added; by unit, lane: states, behind them
    int64_t states;
    int *err;
};

// exp of two log decays, at most 0: above -1/4 as 1 + ld (..), a polynomial of least maximum relative error (6.7e-8, as computed here 1.1e-7) by Lawson's iteration, so that a decay next to 1 is
// rounded to the nearest -- the special-function unit's is not, and a sum over thousands of tokens would show it.  Below, that unit's.
__device__ __forceinline__ f32x2 decay_of(f32x2 ld) {
    f32x2 y = fma2(ld, pack2(0.037709992f, 0.037709992f), pack2(0.16605508f, 0.16605508f));
    y = fma2(y, ld, pack2(0.4999693f, 0.4999693f));
    y = fma2(y, ld, pack2(0.99999976f, 0.99999976f));
    y = fma2(y, ld, pack2(1.f, 1.f));
    float near[2], far[2], l[2];
    unpack2(y, near[0], near[1]);
    unpack2(ld, l[0], l[1]);
    unpack2(mul2(ld, pack2(1.4426950408889634f, 1.4426950408889634f)), far[0], far[1]);
    return pack2(l[0] > -0.25f ? near[0] : ex2_approx(far[0]), l[1] > -0.25f ? near[1] : ex2_approx(far[1]));   // what is not a number stays that
}
// Multipliers of maps, from sums of log decays below zero: exp or, above -1/4, exp - 1, which is below zero.  A map's multiplier next to 1 that is rounded to FP32 would leave a sum
// over many tiles off where decays are all alike (3e-8 a tile); exp - 1 keeps its bits, by a polynomial as above (7.8e-9, as computed here 9.4e-8).
__device__ __forceinline__ f32x2 multiplier(f32x2 ld) {
    f32x2 y = fma2(ld, pack2(0.0075102216f, 0.0075102216f), pack2(0.041488953f, 0.041488953f));
    y = fma2(y, ld, pack2(0.16665082f, 0.16665082f));
    y = fma2(y, ld, pack2(0.4999995f, 0.4999995f));
    y = mul2(fma2(y, ld, pack2(1.f, 1.f)), ld);
    float near[2], far[2], l[2];
    unpack2(y, near[0], near[1]);
    unpack2(ld, l[0], l[1]);
    unpack2(mul2(ld, pack2(1.4426950408889634f, 1.4426950408889634f)), far[0], far[1]);
    return pack2(l[0] > -0.25f ? near[0] : ex2_approx(far[0]), l[1] > -0.25f ? near[1] : ex2_approx(far[1]));
}
// h through a map.  An infinite h comes out as not a number, whatever the map is, and that stays so through all that follow
__device__ __forceinline__ f32x2 through(f32x2 h, f32x2 m, f32x2 x) {
    float ml, mh, kl, kh;
    unpack2(m, ml, mh);
    asm("set.lt.f32.f32 %0, %1, 0f00000000;" : "=f"(kl) : "f"(ml));   // 1 or 0
    asm("set.lt.f32.f32 %0, %1, 0f00000000;" : "=f"(kh) : "f"(mh));
    return fma2(m, h, fma2(pack2(kl, kh), h, x));
}
__device__ __forceinline__ int no_number(f32x2 v) {   // a bit for each of the channels
    float l, h;
    unpack2(v, l, h);
    return (l != l) | (h != h) << 1;
}
// v, or w in the channels of `lost`
__device__ __forceinline__ f32x2 in_place_of(int lost, f32x2 w, f32x2 v) {
    float a[2], b[2];
    unpack2(w, a[0], a[1]);
    unpack2(v, b[0], b[1]);
    return pack2(lost & 1 ? a[0] : b[0], lost & 2 ? a[1] : b[1]);
}
constexpr float GR_BELOW_ZERO = -1e-30f;   // where sums of log decays begin: too small to change one
__device__ __forceinline__ f32x2 held(f32x2 ld) {
    float l, h;
    unpack2(ld, l, h);
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(l) : "f"(0.f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(h) : "f"(0.f));
    return pack2(l, h);
}
__device__ __forceinline__ void tell(unsigned long long *at, f32x2 v) {
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(at), "l"(v == GR_NOTHING ? 0x7fffffff7fffffffull : v) : "memory");
}
__device__ __forceinline__ f32x2 heard(const unsigned long long *at) {
    f32x2 v;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(at) : "memory");
    return v;
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
__global__ void __launch_bounds__(GR_THREADS, BACK ? 2 : 3) recurrence_tiles(const __grid_constant__ RecurrenceKernel p) {
    typedef typename Two<T>::Raw Raw;
    constexpr int ARRAYS = BACK ? 3 : 2, LANES = 128 / sizeof(Raw), RUNS = GR_WARPS * 32 / LANES, RUN = SEQ_TILE / RUNS, CHANNELS = 2 * LANES;
    extern __shared__ unsigned char raw[];
    __shared__ __align__(8) uint64_t bars[GR_STAGES];
    __shared__ f32x2 logs_s[RUNS][LANES], times_s[RUNS][LANES], added_s[RUNS][LANES], enter_s[RUNS][LANES];   // maps of the runs; what enters them
    __shared__ __align__(16) int4 entry_s[GR_STAGES];   // {first row, length, first token, sequence} of a stage's unit
    __shared__ int unit_s[GR_STAGES], gave_up_s;
    const RecurrenceArgs &a = p.a;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const unsigned char *base = raw + (-tc::smem_u32(raw) & 127);
    const uint32_t smem = tc::smem_u32(base), b_full = tc::smem_u32(&bars[0]);
    const f32x2 none = pack2(GR_BELOW_ZERO, GR_BELOW_ZERO);
    if (threadIdx.x == 0) {
        for (int i = 0; i < GR_STAGES; i++) tc::mbar_init(b_full + 8 * i, 1);
        tc::fence_mbar_init();
        gave_up_s = 0;
    }
    __syncthreads();
    const Waits wait{&gave_up_s, p.err};
    // units that the ninth warp's first lane has taken: the next one, known with its entry, and the one behind, asked for
    int next = (int)blockIdx.x, behind = next, copies = 0;
    int4 next_e = make_int4(0, 0, 0, 0);
    auto ask = [&](int u) { return p.counted ? (int)(atomicAdd(p.counter, 1u) + 1u) : u + (int)gridDim.x; };
    auto known = [&](int u) {
        const int i = u / p.groups;
        return u < p.units ? reinterpret_cast<const int4 *>(a.s.table)[seq_by_place(a.s, BACK ? a.s.tiles - 1 - i : i)] : make_int4(0, 0, 0, 0);
    };
    auto start = [&](int stage) {
        unit_s[stage] = min(next, p.units);
        entry_s[stage] = next_e;
        if (next < p.units) {
            tc::mbar_expect_tx(b_full + 8 * stage, ARRAYS * GR_TILE);
            for (int i = 0; i < ARRAYS; i++)   // of the outputs the tokens before
                tc::tma_rows(smem + (ARRAYS * stage + i) * GR_TILE, &p.m[i], next % p.groups * CHANNELS, 0, next_e.x + next_e.z - (i == 2), b_full + 8 * stage);
            copies++;
        }
        next = behind;
        next_e = known(next);
        behind = ask(behind);
    };
    if (threadIdx.x == 32 * GR_WARPS) {
        if (p.counted) next = ask(0);
        next_e = known(next);
        behind = ask(next);
        start(0);
    }
    for (int n = 0;; n++) {
        __syncthreads();   // the unit is known, and all have done with the one before
        const int stage = n % GR_STAGES, u = unit_s[stage];
        if (u >= p.units) break;
        const int4 e = entry_s[stage];
        const int g = u % p.groups;
        if (warp == GR_WARPS) {
            if (lane == 0) start((n + 1) % GR_STAGES);
            __syncwarp();
            const int before = BACK ? (e.y - 1) / SEQ_TILE - e.z / SEQ_TILE : e.z / SEQ_TILE;   // tiles before this one
            const bool last = BACK ? e.z == 0 : e.z + SEQ_TILE >= e.y;
            const int l = lane % LANES, c = g * CHANNELS + 2 * l;
            const float *in = BACK ? a.dstate_out : a.state_in;   // what enters the sequence, and leaves it
            float *out = BACK ? a.dstate_in : a.state_out;
            f32x2 h = 0;
            if (before == 0 && in && c < a.channels) h = *reinterpret_cast<const f32x2 *>(in + (int64_t)e.w * a.channels + c);
            auto run_of = [&](int i) { return BACK ? RUNS - 1 - i : i; };
            unsigned long long *map = p.told + 2 * ((int64_t)u * LANES + l), *state = p.told + p.states + (int64_t)u * LANES + l;
            const int64_t step = (int64_t)p.groups * LANES;
            __syncthreads();   // the runs' maps are there
            f32x2 times = 0, sum = 0;   // the tile's
            int near = 0;               // tiles between this one and the nearest that had told its state
            if (before) {
                if (!last) {
                    f32x2 logs = none;
#pragma unroll 8
                    for (int i = 0; i < RUNS; i++) {
                        logs = add2(logs, logs_s[run_of(i)][l]);
                        sum = through(sum, times_s[run_of(i)][l], added_s[run_of(i)][l]);
                    }
                    times = multiplier(logs);
                    if (lane < LANES) {
                        tell(map, times);
                        tell(map + 1, sum);
                    }
                }
                // a lane looks at one of the 32 tiles before: the nearest that has told its state, with maps told by all in between
                for (uint32_t tries = 0;;) {
                    const bool is = lane < before;
                    const f32x2 s = is ? heard(state - l - (1 + lane) * step) : GR_NOTHING, t = is ? heard(map - 2 * (l + (1 + lane) * step)) : GR_NOTHING;   // its first word
                    const uint32_t has = __ballot_sync(0xffffffffu, s != GR_NOTHING), maps = __ballot_sync(0xffffffffu, t != GR_NOTHING);
                    near = __ffs(has) - 1;
                    bool all = has && (~maps & ((1u << near) - 1)) == 0;
                    if (all) {   // the channels' own words, each of which tells whether it is there
                        h = heard(state - (1 + near) * step);
                        all = h != GR_NOTHING;
#pragma unroll 1
                        for (int d = near; d > 0; d -= GR_MAPS) {   // so many at a time on their way
                            f32x2 t[GR_MAPS], b[GR_MAPS];
#pragma unroll
                            for (int i = 0; i < GR_MAPS; i++)
                                if (d > i) {
                                    t[i] = heard(map - 2 * (d - i) * step);
                                    b[i] = heard(map - 2 * (d - i) * step + 1);
                                }
#pragma unroll
                            for (int i = 0; i < GR_MAPS; i++)
                                if (d > i) {
                                    all &= t[i] != GR_NOTHING && b[i] != GR_NOTHING;
                                    h = through(h, t[i], b[i]);
                                }
                        }
                    }
                    if (__all_sync(0xffffffffu, all)) break;
                    if (__any_sync(0xffffffffu, gave_up_s) || ++tries > 2 * WAIT_TRIES) {   // a try takes half a microsecond or more
                        if (lane == 0) {
                            gave_up_s = 1;
                            *(volatile int *)p.err = 1;
                        }
                        break;
                    }
                }
            }
            const bool told = before && !last && lane < LANES;
            const f32x2 own = through(h, times, sum);   // through the tile's own map, as those do who look over it
            if (told && !no_number(own)) tell(state, own);
            f32x2 leaves = h;
#pragma unroll 8
            for (int i = 0; i < RUNS; i++) {
                if (lane < LANES) enter_s[run_of(i)][l] = leaves;
                leaves = through(leaves, times_s[run_of(i)][l], added_s[run_of(i)][l]);
            }
            if (const int lost = no_number(leaves) | no_number(own)) {
                // Something was infinite here, or is not a number: maps do not tell which.  What enters is then what the tile before tells, which is waited for (unless there was
                // no number farther back already), and goes through the tile token by token, as the definition has it.  65536 tokens with an infinite one in front: 2 ms.
                if (before) {
                    f32x2 from = heard(state - (1 + near) * step);
                    if (near && (no_number(h) & ~no_number(from)))
                        for (uint32_t tries = 0; (from = heard(state - step)) == GR_NOTHING && !*(volatile int *)&gave_up_s;)
                            if (++tries > 2 * WAIT_TRIES) {
                                gave_up_s = 1;
                                *(volatile int *)p.err = 1;
                            }
                    h = in_place_of(no_number(h), from, h);
                }
                if (lost & ~no_number(h)) {
                    wait(b_full + 8 * stage, (n / GR_STAGES) & 1);
                    const unsigned char *tile = base + ARRAYS * stage * GR_TILE + l * sizeof(Raw);
                    const int count = min(SEQ_TILE, e.y - e.z);
#pragma unroll 8
                    for (int k = 0; k < SEQ_TILE; k++) {
                        const int i = BACK ? SEQ_TILE - 1 - k : k;
                        if (k % RUN == 0 && lane < LANES) enter_s[i / RUN][l] = in_place_of(no_number(enter_s[i / RUN][l]), h, enter_s[i / RUN][l]);
                        const f32x2 m = decay_of(held(Two<T>::open(*reinterpret_cast<const Raw *>(tile + GR_TILE + i * 128)))), x = Two<T>::open(*reinterpret_cast<const Raw *>(tile + i * 128));
                        if (i < count) h = BACK ? mul2(m, add2(h, x)) : fma2(m, h, x);
                    }
                    leaves = in_place_of(no_number(leaves), h, leaves);
                }
                if (told) tell(state, in_place_of(lost, leaves, own));
            }
            __syncthreads();   // what enters the runs is there
            if (last) {
                if (out && lane < LANES && c < a.channels) *reinterpret_cast<f32x2 *>(out + (int64_t)e.w * a.channels + c) = leaves;
            } else if (before == 0 && lane < LANES) {
                tell(state, leaves);
            }
        } else {
            const int run = warp * (32 / LANES) + lane / LANES, l = lane % LANES, r0 = run * RUN, c = g * CHANNELS + 2 * l, count = min(SEQ_TILE, e.y - e.z) - r0;
            const unsigned char *tile = base + ARRAYS * stage * GR_TILE + r0 * 128 + l * sizeof(Raw);
            auto raw_of = [&](int array, int i) { return *reinterpret_cast<const Raw *>(tile + array * GR_TILE + i * 128); };
            f32x2 m[RUN], logs = none, sum = 0;
            wait(b_full + 8 * stage, (n / GR_STAGES) & 1);
            auto first = [&](auto whole) {   // whether all of the run's tokens are the sequence's
                const bool all = decltype(whole)::value;
#pragma unroll
                for (int k = 0; k < RUN; k++) {
                    const int i = BACK ? RUN - 1 - k : k;
                    const f32x2 ld = all || i < count ? held(Two<T>::open(raw_of(1, i))) : 0ull, x = all || i < count ? Two<T>::open(raw_of(0, i)) : 0ull;   // x, or dout
                    m[i] = decay_of(ld);
                    logs = add2(logs, ld);
                    sum = BACK ? mul2(m[i], add2(sum, x)) : fma2(m[i], sum, x);
                }
            };
            if (count >= RUN) first(std::true_type());
            else first(std::false_type());
            logs_s[run][l] = logs;
            times_s[run][l] = multiplier(logs);
            added_s[run][l] = sum;
            __syncthreads();   // the runs' maps are there
            const int64_t t0 = (int64_t)e.x + e.z + r0;
            T *y = reinterpret_cast<T *>(BACK ? a.dx.data : a.out.data) + t0 * (BACK ? a.dx.token_stride : a.out.token_stride) + c;
            T *z = BACK ? reinterpret_cast<T *>(a.dlog_decay.data) + t0 * a.dlog_decay.token_stride + c : nullptr;
            const bool in = c < a.channels;
            __syncthreads();   // what enters the runs is there
            f32x2 h = enter_s[run][l];
            auto second = [&](auto whole) {
                const bool all = decltype(whole)::value;
#pragma unroll
                for (int k = 0; k < RUN; k++) {
                    const int i = BACK ? RUN - 1 - k : k;
                    if (!all && i >= count) continue;
                    const f32x2 x = Two<T>::open(raw_of(0, i));
                    if constexpr (!BACK) {
                        h = fma2(m[i], h, x);
                        if (in) *reinterpret_cast<Raw *>(y + i * a.out.token_stride) = Two<T>::close(h);
                    } else {
                        const f32x2 d = add2(h, x);
                        h = mul2(m[i], d);
                        f32x2 past = Two<T>::open(raw_of(2, i));   // as rounded in `out`: half a step of the type in dlog_decay, and no second walk forward
                        if (i == 0 && e.z + r0 == 0) past = a.state_in && in ? *reinterpret_cast<const f32x2 *>(a.state_in + (int64_t)e.w * a.channels + c) : 0;
                        float ll, lh, dl, dh;
                        unpack2(Two<T>::open(raw_of(1, i)), ll, lh);
                        unpack2(mul2(h, past), dl, dh);
                        if (!in) continue;
                        *reinterpret_cast<Raw *>(y + i * a.dx.token_stride) = Two<T>::close(d);
                        *reinterpret_cast<Raw *>(z + i * a.dlog_decay.token_stride) = Two<T>::close(pack2(ll > 0.f ? 0.f : dl, lh > 0.f ? 0.f : dh));
                    }
                }
            };
            if (count >= RUN) second(std::true_type());
            else second(std::false_type());
        }
    }
    if (threadIdx.x == 32 * GR_WARPS)   // copies that nobody waited for, where the block gave up
        for (int i = max(0, copies - GR_STAGES); i < copies; i++) wait.drain(b_full + 8 * (i % GR_STAGES), (i / GR_STAGES) & 1);
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

// the counter, and two words of maps and one of states by tile and lane
static size_t lane_places(const f3m_seqs &s, int channels) { return (size_t)s.tiles * ((channels + 63) / 64) * 32; }
size_t recurrence_workspace(const f3m_seqs &s, int channels) { return s.longest > SEQ_TILE ? 16 + lane_places(s, channels) * 24 : 0; }

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
    p.groups = (a.channels + channels - 1) / channels;
    F3M_REQUIRE((int64_t)a.s.tiles * p.groups <= 0x7fff0000, F3M_ERR_OVERFLOW, "%d tiles of %d channels do not fit in 31 bits", a.s.tiles, a.channels);
    p.units = a.s.tiles * p.groups;
    p.counted = a.s.longest > SEQ_TILE;
    p.counter = reinterpret_cast<unsigned *>(a.ws);
    p.told = reinterpret_cast<unsigned long long *>(reinterpret_cast<char *>(a.ws) + 16);
    p.states = 2 * (int64_t)lane_places(a.s, a.channels);
    p.err = seq_error_word();
    p.m[0] = channel_tensor_map(type, BACK ? a.dout : a.x, a.s.tokens, a.channels);
    p.m[1] = channel_tensor_map(type, a.log_decay, a.s.tokens, a.channels);
    if (BACK) p.m[2] = channel_tensor_map(type, a.out, a.s.tokens, a.channels);
    if (p.counted) F3M_CUDA(cudaMemsetAsync(a.ws, 0xff, recurrence_workspace(a.s, a.channels), s));
    const int bytes = GR_STAGES * (BACK ? 3 : 2) * GR_TILE + 128;
    static SharedMemory allowed;
    allowed.allow(recurrence_tiles<T, BACK>, bytes);
    recurrence_tiles<T, BACK><<<std::min(p.units, (BACK ? 2 : 3) * NUM_SMS_HINT), GR_THREADS, bytes, s>>>(p);
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
