// extern "C" entry points of the kernel products over sequences: checks of the arguments, the table of tiles, workspaces.
#include <algorithm>
#include <exception>
#include <numeric>
#include "seq.cuh"

namespace f3m {

int *seq_error_word() {
    static int *word = [] {   // once per process, possibly while a stream is being captured
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        cudaThreadExchangeStreamCaptureMode(&mode);
        int *p = nullptr;
        const cudaError_t e = cudaHostAlloc((void **)&p, 64, cudaHostAllocMapped | cudaHostAllocPortable);
        cudaThreadExchangeStreamCaptureMode(&mode);
        F3M_REQUIRE(e == cudaSuccess, F3M_ERR_CUDA, "cudaHostAlloc failed: %s", cudaGetErrorString(e));
        *p = 0;
        return p;
    }();
    return word;
}
void seq_check_error() {
    volatile int *w = seq_error_word();
    if (*w) {
        *w = 0;
        F3M_REQUIRE(false, F3M_ERR_INTERNAL, "a kernel of an earlier call on sequences gave up waiting: that call's outputs are not valid");
    }
}

CUtensorMap seq_tensor_map(int type, const f3m_rows &r, int64_t tokens, int heads, int width) {
    typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                               const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        F3M_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found));
        F3M_REQUIRE(f && found == cudaDriverEntryPointSuccess, F3M_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        return (Encode)f;
    }();
    CUtensorMap m;
    const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)tokens}, strides[2] = {2ull * r.head_stride, 2ull * r.token_stride};
    const cuuint32_t box[3] = {64, 1, SEQ_TILE}, step[3] = {1, 1, 1};
    const CUresult e = encode(&m, type == F3M_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, r.data, dims, strides, box, step,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    F3M_REQUIRE(e == CUDA_SUCCESS, F3M_ERR_ARG, "no tensor map for %lld tokens, %d heads, width %d, strides %lld, %lld (driver error %d)", (long long)tokens, heads,
                width, (long long)r.token_stride, (long long)r.head_stride, (int)e);
    return m;
}

}  // namespace f3m

using namespace f3m;

namespace {

template <typename F>
int guarded(F &&f) {
    try {
        set_error("%s", "");
        f();
        return F3M_OK;
    } catch (const Fail &e) {
        return e.code;
    } catch (const std::exception &e) {
        set_error("%s", e.what());
        return F3M_ERR_INTERNAL;
    }
}

void check_type(int type) {
    F3M_REQUIRE(type == F3M_TYPE_BF16 || type == F3M_TYPE_F16, F3M_ERR_UNSUPPORTED, "type %d: only bf16 and fp16 are built", type);
}
void check_width(int w, const char *what) {
    F3M_REQUIRE(w >= 8 && w <= F3M_MAX_WIDTH && w % 8 == 0, F3M_ERR_UNSUPPORTED, "%s %d is not a multiple of 8 in 8..%d", what, w, F3M_MAX_WIDTH);
}
void check_heads(int heads, int kv_heads) {
    F3M_REQUIRE(heads >= 1 && heads <= 65535 && kv_heads >= 1 && heads % kv_heads == 0, F3M_ERR_ARG, "%d heads do not share %d key heads evenly", heads, kv_heads);
}
void check_seqs(const f3m_seqs *s) {
    F3M_REQUIRE(s, F3M_ERR_ARG, "null pointer argument");
    F3M_REQUIRE(s->sequences >= 0 && s->tiles >= 0 && s->pairs >= 0 && s->tokens >= 0 && s->tokens <= F3M_SEQ_MAX_TOKENS, F3M_ERR_ARG, "counts of the sequences were not filled by f3m_seqs_layout");
    F3M_REQUIRE(s->sequences == 0 || (s->table && (uintptr_t)s->table % 16 == 0), F3M_ERR_ARG, "the table of the sequences is missing or not 16-byte aligned");
}
// tokens == 0: the array may be absent
void check_rows(const f3m_rows &r, int64_t tokens, int heads, int width, const char *what) {
    if (tokens == 0) return;
    F3M_REQUIRE(r.data, F3M_ERR_ARG, "%s: null pointer", what);
    F3M_REQUIRE((uintptr_t)r.data % 16 == 0, F3M_ERR_ARG, "%s does not start on 16 bytes", what);
    F3M_REQUIRE(r.token_stride % 8 == 0 && r.head_stride % 8 == 0 && r.token_stride >= 0 && r.head_stride >= 0 && r.token_stride < ((int64_t)1 << 36) &&
                    r.head_stride < ((int64_t)1 << 36),
                F3M_ERR_ARG, "%s: strides %lld, %lld are not multiples of 8 elements", what, (long long)r.token_stride, (long long)r.head_stride);
}
// an output's elements have to be different places
void check_out(const f3m_rows &r, int64_t tokens, int heads, int width, const char *what) {
    check_rows(r, tokens, heads, width, what);
    if (tokens == 0) return;
    const int64_t a = std::min(r.token_stride, r.head_stride), b = std::max(r.token_stride, r.head_stride);
    const int64_t n = r.token_stride <= r.head_stride ? tokens : heads;
    const bool one = tokens == 1 || heads == 1;   // one axis only: the other stride is not used
    const int64_t used = tokens == 1 ? r.head_stride : r.token_stride;
    F3M_REQUIRE(one ? ((tokens == 1 && heads == 1) || used >= width) : (a >= width && b >= a * (n - 1) + width), F3M_ERR_ARG,
                "%s: rows overlap (strides %lld, %lld)", what, (long long)r.token_stride, (long long)r.head_stride);
}
void check_window(int window, int sinks, float scale) {
    F3M_REQUIRE(window >= 1 && sinks >= 0, F3M_ERR_ARG, "window %d, sinks %d: at least one key is seen", window, sinks);
    F3M_REQUIRE(isfinite(scale), F3M_ERR_ARG, "scale is not finite");
}
void check_workspace(const void *ws, size_t have, size_t need) {
    F3M_REQUIRE(need == 0 || (ws && (uintptr_t)ws % 16 == 0), F3M_ERR_ARG, "the workspace is missing or not 16-byte aligned");
    F3M_REQUIRE(have >= need, F3M_ERR_TOO_LARGE, "the workspace of %zu bytes is too small: %zu bytes are needed", have, need);
}
void check_state(const float *p, const char *what) { F3M_REQUIRE((uintptr_t)p % 16 == 0, F3M_ERR_ARG, "%s is not 16-byte aligned", what); }

}  // namespace

extern "C" {

int f3m_seqs_layout(const int32_t *lengths, int32_t n, f3m_seqs *seqs, int32_t *table) {
    return guarded([&] {
        F3M_REQUIRE(seqs && n >= 0 && (lengths || n == 0), F3M_ERR_ARG, "bad argument to f3m_seqs_layout");
        int64_t tokens = 0, tiles = 0, pairs = 0;
        int32_t longest = 0, empty = 0;
        for (int i = 0; i < n; i++) {
            F3M_REQUIRE(lengths[i] >= 0, F3M_ERR_ARG, "length %d of sequence %d", lengths[i], i);
            tokens += lengths[i];
            tiles += ((int64_t)lengths[i] + SEQ_TILE - 1) / SEQ_TILE;
            pairs += ((int64_t)lengths[i] + 2 * SEQ_TILE - 1) / (2 * SEQ_TILE);
            longest = std::max(longest, lengths[i]);
            empty += lengths[i] == 0;
        }
        F3M_REQUIRE(tokens <= F3M_SEQ_MAX_TOKENS, F3M_ERR_OVERFLOW, "%lld tokens do not fit in 31 bits", (long long)tokens);
        F3M_REQUIRE(4 * (3 * tiles + n + pairs) <= 0x7fffffff, F3M_ERR_OVERFLOW, "the table of %d sequences does not fit in 31 bits", n);
        seqs->table = nullptr;
        seqs->tokens = tokens;
        seqs->sequences = n;
        seqs->tiles = (int32_t)tiles;
        seqs->longest = longest;
        seqs->empty = empty;
        seqs->pairs = (int32_t)pairs;
        seqs->table_words = (int32_t)(4 * (3 * tiles + n + pairs));
        if (!table) return;
        int32_t *t = table, *sq = table + 12 * tiles;
        int32_t first = 0, tile = 0;
        for (int i = 0; i < n; i++) {
            const int32_t len = lengths[i], nt = (int32_t)(((int64_t)len + SEQ_TILE - 1) / SEQ_TILE);
            sq[4 * i] = first; sq[4 * i + 1] = len; sq[4 * i + 2] = tile; sq[4 * i + 3] = nt;
            for (int32_t k = 0; k < nt; k++, t += 4) { t[0] = first; t[1] = len; t[2] = k * SEQ_TILE; t[3] = i; }
            first += len;
            tile += nt;
        }
        std::vector<int32_t> order((size_t)tiles);
        for (int which = 1; which <= 2; which++) {
            std::iota(order.begin(), order.end(), 0);
            std::stable_sort(order.begin(), order.end(), [&](int32_t x, int32_t y) {
                const int32_t *a = table + 4 * (size_t)x, *b = table + 4 * (size_t)y;
                return which == 1 ? a[2] > b[2] : a[1] - a[2] > b[1] - b[2];
            });
            for (int64_t k = 0; k < tiles; k++) memcpy(table + 4 * (which * tiles + k), table + 4 * (size_t)order[k], 16);
        }
        int32_t *pr = sq + 4 * (int64_t)n;
        for (int64_t k = tiles; k < 2 * tiles; k++)
            if (table[4 * k + 2] / SEQ_TILE % 2 == 0) { memcpy(pr, table + 4 * k, 16); pr += 4; }
    });
}

int *f3m_seqs_error_word(void) {
    int *word = nullptr;
    guarded([&] { word = seq_error_word(); });
    return word;
}

int f3m_window_attention(const f3m_seqs *seqs, int32_t type, int32_t heads, int32_t kv_heads, int32_t width, int32_t window, int32_t sinks,
                         float scale, f3m_rows q, f3m_rows k, f3m_rows v, f3m_rows out, float *lse, void *stream) {
    return guarded([&] {
        check_seqs(seqs); check_type(type); check_heads(heads, kv_heads); check_width(width, "width"); check_window(window, sinks, scale);
        const int64_t n = seqs->tokens;
        check_rows(q, n, heads, width, "q"); check_rows(k, n, kv_heads, width, "k"); check_rows(v, n, kv_heads, width, "v");
        check_out(out, n, heads, width, "out");
        F3M_REQUIRE(n == 0 || lse, F3M_ERR_ARG, "lse: null pointer");
        if (n == 0) return;
        seq_check_error();
        WindowArgs a{*seqs, heads, kv_heads, width, window, sinks, scale, q, k, v, out, lse};
        window_forward(type, a, (cudaStream_t)stream);
    });
}

size_t f3m_window_attention_grad_workspace_bytes(const f3m_seqs *seqs, int32_t heads, int32_t kv_heads, int32_t width, int32_t window, int32_t sinks) {
    if (!seqs || seqs->tokens <= 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || width < 8 || window < 1 || sinks < 0) return 0;
    return window_grad_workspace(*seqs, heads, kv_heads, width, window, sinks);
}

int f3m_window_attention_grad(const f3m_seqs *seqs, int32_t type, int32_t heads, int32_t kv_heads, int32_t width, int32_t window, int32_t sinks,
                              float scale, f3m_rows q, f3m_rows k, f3m_rows v, f3m_rows out, const float *lse, f3m_rows dout, f3m_rows dq,
                              f3m_rows dk, f3m_rows dv, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        check_seqs(seqs); check_type(type); check_heads(heads, kv_heads); check_width(width, "width"); check_window(window, sinks, scale);
        const int64_t n = seqs->tokens;
        check_rows(q, n, heads, width, "q"); check_rows(k, n, kv_heads, width, "k"); check_rows(v, n, kv_heads, width, "v");
        check_rows(out, n, heads, width, "out"); check_rows(dout, n, heads, width, "dout");
        check_out(dq, n, heads, width, "dq"); check_out(dk, n, kv_heads, width, "dk"); check_out(dv, n, kv_heads, width, "dv");
        F3M_REQUIRE(n == 0 || lse, F3M_ERR_ARG, "lse: null pointer");
        if (n == 0) return;
        check_workspace(workspace, workspace_bytes, window_grad_workspace(*seqs, heads, kv_heads, width, window, sinks));
        seq_check_error();
        WindowArgs a{*seqs, heads, kv_heads, width, window, sinks, scale, q, k, v, out, const_cast<float *>(lse), dout, dq, dk, dv, (float *)workspace};
        window_backward(type, a, (cudaStream_t)stream);
    });
}

static bool step_sizes(int32_t n, int32_t heads, int32_t kv_heads, int32_t width, int64_t capacity, int32_t window, int32_t sinks) {
    return n > 0 && heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && width >= 8 && width <= F3M_MAX_WIDTH && capacity > 0 && window >= 1 && sinks >= 0;
}

size_t f3m_window_attention_step_workspace_bytes(int32_t n, int32_t heads, int32_t kv_heads, int32_t width, int64_t capacity, int32_t window,
                                                 int32_t sinks) {
    if (!step_sizes(n, heads, kv_heads, width, capacity, window, sinks)) return 0;
    return window_step_part_floats(n, heads, width, window_step_parts(n, heads, kv_heads, capacity, window, sinks)) * sizeof(float);
}

int f3m_window_attention_step(int32_t n, int32_t type, int32_t heads, int32_t kv_heads, int32_t width, int64_t capacity, int32_t window,
                              int32_t sinks, float scale, f3m_rows q, f3m_rows k_cache, int64_t k_seq_stride, f3m_rows v_cache,
                              int64_t v_seq_stride, const int32_t *lengths, f3m_rows out, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        check_type(type); check_heads(heads, kv_heads); check_width(width, "width"); check_window(window, sinks, scale);
        F3M_REQUIRE(n >= 0 && capacity >= 0 && capacity <= F3M_SEQ_MAX_TOKENS, F3M_ERR_ARG, "%d sequences of capacity %lld", n, (long long)capacity);
        check_rows(q, n, heads, width, "q"); check_out(out, n, heads, width, "out");
        check_rows(k_cache, n ? capacity : 0, kv_heads, width, "k_cache"); check_rows(v_cache, n ? capacity : 0, kv_heads, width, "v_cache");
        F3M_REQUIRE(k_seq_stride % 8 == 0 && v_seq_stride % 8 == 0 && k_seq_stride >= 0 && v_seq_stride >= 0, F3M_ERR_ARG, "strides of the cache's sequences are not multiples of 8 elements");
        F3M_REQUIRE(n == 0 || lengths, F3M_ERR_ARG, "lengths: null pointer");
        if (n == 0) return;
        StepArgs a{n, heads, kv_heads, width, window, sinks, capacity, scale, q, k_cache, v_cache, out, k_seq_stride, v_seq_stride, lengths, 1, (float *)workspace};
        a.parts = window_step_parts(n, heads, kv_heads, capacity, window, sinks);
        check_workspace(workspace, workspace_bytes, window_step_part_floats(n, heads, width, a.parts) * sizeof(float));
        seq_check_error();
        window_step(type, a, (cudaStream_t)stream);
    });
}

size_t f3m_decay_attention_workspace_bytes(const f3m_seqs *seqs, int32_t heads, int32_t width_k, int32_t width_v) {
    return seqs && heads > 0 && width_k > 0 && width_v > 0 ? decay_workspace(*seqs, heads, width_k, width_v) : 0;
}

static void check_decay(const f3m_seqs *seqs, int type, int heads, int width_k, int width_v, const float *log_decay, float scale) {
    check_seqs(seqs); check_type(type); check_heads(heads, heads); check_width(width_k, "width_k"); check_width(width_v, "width_v");
    F3M_REQUIRE(log_decay || seqs->sequences == 0, F3M_ERR_ARG, "log_decay: null pointer");
    F3M_REQUIRE(isfinite(scale), F3M_ERR_ARG, "scale is not finite");
}

int f3m_decay_attention(const f3m_seqs *seqs, int32_t type, int32_t heads, int32_t width_k, int32_t width_v, const float *log_decay, float scale,
                        f3m_rows q, f3m_rows k, f3m_rows v, const float *state_in, f3m_rows out, float *state_out, void *workspace,
                        size_t workspace_bytes, void *stream) {
    return guarded([&] {
        check_decay(seqs, type, heads, width_k, width_v, log_decay, scale);
        const int64_t n = seqs->tokens;
        check_rows(q, n, heads, width_k, "q"); check_rows(k, n, heads, width_k, "k"); check_rows(v, n, heads, width_v, "v");
        check_out(out, n, heads, width_v, "out");
        check_state(state_in, "state_in"); check_state(state_out, "state_out");
        F3M_REQUIRE(!state_in || state_in != state_out, F3M_ERR_ARG, "state_in and state_out are the same array");
        check_workspace(workspace, workspace_bytes, decay_workspace(*seqs, heads, width_k, width_v));
        if (seqs->sequences == 0) return;
        seq_check_error();
        decay_product(type, DecayArgs{*seqs, heads, width_k, width_v, log_decay, scale, 1.f, false, false, false, q, k, v, out, state_in, state_out, workspace}, (cudaStream_t)stream);
    });
}

int f3m_decay_attention_grad(const f3m_seqs *seqs, int32_t type, int32_t heads, int32_t width_k, int32_t width_v, const float *log_decay,
                             float scale, f3m_rows q, f3m_rows k, f3m_rows v, const float *state_in, f3m_rows dout, const float *dstate_out,
                             f3m_rows dq, f3m_rows dk, f3m_rows dv, float *dstate_in, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded([&] {
        check_decay(seqs, type, heads, width_k, width_v, log_decay, scale);
        const int64_t n = seqs->tokens;
        check_rows(q, n, heads, width_k, "q"); check_rows(k, n, heads, width_k, "k"); check_rows(v, n, heads, width_v, "v");
        check_rows(dout, n, heads, width_v, "dout");
        check_out(dq, n, heads, width_k, "dq"); check_out(dk, n, heads, width_k, "dk"); check_out(dv, n, heads, width_v, "dv");
        check_state(state_in, "state_in"); check_state(dstate_out, "dstate_out"); check_state(dstate_in, "dstate_in");
        F3M_REQUIRE(!dstate_out || dstate_out != dstate_in, F3M_ERR_ARG, "dstate_out and dstate_in are the same array");
        check_workspace(workspace, workspace_bytes, decay_workspace(*seqs, heads, width_k, width_v));
        if (seqs->sequences == 0) return;
        seq_check_error();
        // dq_i = scale sum_(j <= i) decay^(i-j) (dout_i.v_j) k_j + scale decay^(i+1) S dout_i: the product itself with (dout, v, k), state
        // transposed.  dk and dv come from the adjoint recurrence D_t = scale q_t dout_t^T + decay D_(t+1), dk_t = D_t v_t, dv_t = D_t^T k_t:
        // the product from the end with (v, dout, q) and (k, q, dout).
        // The two have one state, to a transposition: what lies between the ranges is computed once.
        decay_product(type, DecayArgs{*seqs, heads, width_k, width_v, log_decay, 1.f, scale, true, false, false, k, q, dout, dv, dstate_out, dstate_in, workspace}, (cudaStream_t)stream);
        decay_product(type, DecayArgs{*seqs, heads, width_v, width_k, log_decay, 1.f, scale, true, true, true, v, dout, q, dk, dstate_out, nullptr, workspace}, (cudaStream_t)stream);
        decay_product(type, DecayArgs{*seqs, heads, width_v, width_k, log_decay, scale, 1.f, false, true, false, dout, v, k, dq, state_in, nullptr, workspace}, (cudaStream_t)stream);
    });
}

int f3m_decay_attention_step(int32_t n, int32_t type, int32_t heads, int32_t width_k, int32_t width_v, const float *log_decay, float scale,
                             f3m_rows q, f3m_rows k, f3m_rows v, float *state, f3m_rows out, void *stream) {
    return guarded([&] {
        check_type(type); check_heads(heads, heads); check_width(width_k, "width_k"); check_width(width_v, "width_v");
        F3M_REQUIRE(n >= 0 && (n == 0 || (log_decay && state)), F3M_ERR_ARG, "null pointer argument");
        F3M_REQUIRE(isfinite(scale), F3M_ERR_ARG, "scale is not finite");
        check_rows(q, n, heads, width_k, "q"); check_rows(k, n, heads, width_k, "k"); check_rows(v, n, heads, width_v, "v");
        check_out(out, n, heads, width_v, "out"); check_state(state, "state");
        if (n == 0) return;
        seq_check_error();
        decay_step(type, n, heads, width_k, width_v, log_decay, scale, q, k, v, state, out, (cudaStream_t)stream);
    });
}

}  // extern "C"
