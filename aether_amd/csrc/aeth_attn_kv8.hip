// Attention over the 8-bit cache for a sequence, a chunk of it, and a batch: launches and entry points. The mathematics and the
// kernels: aeth_attn_kv8_dev.hpp.
#include "aeth_attn_kv8_dev.hpp"

int64_t aeth_attn_kv8_ws(int64_t seqs, int64_t n, int64_t nq, int64_t nkv, int64_t hd, int64_t len) {
    if (len <= 4 * KV8_TILE) return 0;  // never split
    // `units` column blocks are split into at most target / units + 1 chunks each, or not at all: fewer than
    // 2·target partials, and target + units. A smaller call (fewer sequences or queries) may take another form.
    const int64_t cols = n * (nq / nkv), cus = aeth_num_cus();
    auto need = [&](int64_t cw, int64_t target) {
        const int64_t units = seqs * nkv * aeth_cdiv(cols, cw);
        return (target + std::min(units, target)) * cw;
    };
    int64_t most = need(16, 4 * cus);
    if (hd <= 128 && cols > 64) most = std::max(most, need(128, 2 * cus));
    if (hd == 128 && cols > 64) most = std::max(most, need(256, cus));
    return most * (hd + 2) * (int64_t)sizeof(float);
}

int aeth_attn_kv8_launch(const float* q, int64_t q_stride, const void* cache, int64_t seq_bytes, const int* lens, int len_add,
                         int64_t seqs, int64_t n, int64_t nq, int64_t nkv, int64_t hd, int64_t max_seq, int64_t max_len,
                         int64_t window, float* out, void* ws, hipStream_t s) {
    if (n <= 0 || seqs <= 0) return AETH_OK;
    A8 A = a8_args(q, q_stride, cache, seq_bytes, lens, len_add, n, nq, nkv, max_seq, max_len, window, out, ws);
    const Form f = a8_form(seqs, n, A.G, nkv, hd, max_len, A.window, lens != nullptr);
    a8_take(A, f);
    if (hd == 64) return a8_launch<64, 0>(A, f, seqs, s);
    if (hd == 128) return a8_launch<128, 0>(A, f, seqs, s);
    return a8_launch<256, 0>(A, f, seqs, s);
}

int aeth_attn_kv8_step_launch(const float* qkv, int64_t nq, int64_t nkv, int64_t hd, const int* st, const float* sin_t,
                              const float* cos_t, int64_t max_seq, int64_t window, void* cache, float* out, void* ws, hipStream_t s) {
    const int64_t G = nq / nkv;
    if (hd != 128 || G > 16 || (((uintptr_t)qkv | (uintptr_t)out | (uintptr_t)sin_t | (uintptr_t)cos_t) & 15))
        return aeth_set_error(AETH_EUNSUPPORTED, "8-bit cache step: %lld heads of %lld a KV head", (long long)G, (long long)hd);
    A8 A = {};
    A.q = qkv;
    A.q_stride = nq * hd;
    A.cache = (const uint8_t*)cache;
    A.lens = st + 2;
    A.len_add = 1;
    A.max_len = (int)max_seq;
    A.n = 1;
    A.nq = (int)nq;
    A.nkv = (int)nkv;
    A.G = A.cols = (int)G;
    A.tiles = (int)aeth_cdiv(max_seq, KV8_TILE);
    A.window = window > 0 && window < max_seq ? (int)window : 0;
    A.out = out;
    A.ws = (float*)ws;
    A.qvec = A.ovec = 1;
    A.pos = st + 1;
    A.sin_t = sin_t;
    A.cos_t = cos_t;
    A.max_seq = max_seq;
    const Form f = a8_form(1, 1, G, nkv, hd, max_seq, A.window, true);
    A.ncb = 1;
    A.tpc = f.tpc;
    A.chunks = f.chunks;
    hipLaunchKernelGGL((k_attn8<128, A8_STEP>), dim3((unsigned)nkv, 1, (unsigned)A.chunks), dim3(256), 0, s, A);
    AETH_LAUNCH_CHECK();
    if (A.chunks > 1) {
        a8_merge<128, 0>(A, 16, 1, s);
        AETH_LAUNCH_CHECK();
    }
    return AETH_OK;
}

int aeth_attn_kv8_check(const char* what, const float* q, int64_t q_stride, const void* cache, int64_t seqs, int64_t n, int64_t nq,
                        int64_t nkv, int64_t hd, int64_t max_seq, int64_t max_len, int64_t window, const float* out, const void* ws) {
    if (!q || !cache || !out || ((uintptr_t)cache & 15) || (((uintptr_t)q | (uintptr_t)out) & 3) || ((uintptr_t)ws & 15))
        return aeth_set_error(AETH_EINVAL, "%s: bad argument (cache and workspace 16-byte aligned, rows 4-byte)", what);
    if (nkv <= 0 || nq <= 0 || nq % nkv != 0 || max_seq <= 0 || max_seq > KV8_MAX_SEQ || window < 0 || n < 0 || seqs < 0)
        return aeth_set_error(AETH_EINVAL, "%s: bad shape (heads %lld / %lld, max_seq %lld, window %lld)", what, (long long)nq,
                              (long long)nkv, (long long)max_seq, (long long)window);
    if (!aeth_kv8_head_dim(hd) || nq > 4096)
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld heads of %lld (head_dim 64, 128 or 256)", what, (long long)nq, (long long)hd);
    if (max_len < n || max_len > max_seq)
        return aeth_set_error(AETH_EINVAL, "%s: %lld queries, %lld of %lld positions", what, (long long)n, (long long)max_len, (long long)max_seq);
    int64_t span;
    if ((n > 1 || seqs > 1) ? (q_stride < nq * hd || !aeth_mul_ok(seqs * n, q_stride, &span) || span > INT64_MAX / 4) : q_stride < 0)
        return aeth_set_error(AETH_EINVAL, "%s: query stride %lld of rows of %lld", what, (long long)q_stride, (long long)(nq * hd));
    if (n * nq > (int64_t)1 << 24 || seqs > 65535 || seqs * n * nq > (int64_t)1 << 28)
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld x %lld queries of %lld heads in one call", what, (long long)seqs, (long long)n, (long long)nq);
    return AETH_OK;
}

int aeth_attn_kv8_check_ws(const char* what, const void* ws, int64_t ws_bytes, int64_t need) {
    if (need > 0 && (!ws || ws_bytes < need))
        return aeth_set_error(AETH_EINVAL, "%s: a workspace of %lld bytes (%lld given)", what, (long long)need, (long long)(ws ? ws_bytes : 0));
    return AETH_OK;
}

int aeth_attn_kv8_check_slices(const char* what, int64_t n_seqs, int64_t layer_stride, int64_t nkv, int64_t hd, int64_t max_seq) {
    int64_t all;
    if (layer_stride < 0 || (layer_stride & 15) || !aeth_mul_ok(n_seqs, layer_stride, &all) ||
        (n_seqs > 1 && layer_stride < nkv * aeth_cdiv(max_seq, KV8_TILE) * aeth_kv8_tile_bytes((int)hd)))
        return aeth_set_error(AETH_EINVAL, "%s: %lld sequences %lld bytes apart", what, (long long)n_seqs, (long long)layer_stride);
    return AETH_OK;
}

extern "C" AETH_API int64_t aeth_attn_kv8_ws_bytes(int64_t n_seqs, int64_t n, int64_t n_heads, int64_t kv_heads, int64_t head_dim,
                                                   int64_t max_len) {
    if (n_seqs < 0 || n < 0 || kv_heads <= 0 || n_heads <= 0 || n_heads % kv_heads != 0 || n_heads > 4096 || !aeth_kv8_head_dim(head_dim) ||
        max_len < 0 || max_len > KV8_MAX_SEQ || n_seqs > 65535 || n > (int64_t)1 << 24) {
        aeth_set_error(AETH_EINVAL, "aeth_attn_kv8_ws_bytes: bad shape");
        return -1;
    }
    return aeth_attn_kv8_ws(n_seqs, n, n_heads, kv_heads, head_dim, max_len);
}

extern "C" AETH_API int aeth_attn_kv8(const float* d_q, int64_t q_stride, const void* d_layer, int64_t n, int64_t n_heads,
                                      int64_t kv_heads, int64_t head_dim, int64_t max_seq, int64_t seq, int64_t window,
                                      float* d_out, void* d_ws, int64_t ws_bytes, void* stream) {
    const char* what = "aeth_attn_kv8";
    int rc = aeth_attn_kv8_check(what, d_q, q_stride, d_layer, 1, n, n_heads, kv_heads, head_dim, max_seq, seq, window, d_out, d_ws);
    if (!rc) rc = aeth_attn_kv8_check_ws(what, d_ws, ws_bytes, aeth_attn_kv8_ws(1, n, n_heads, kv_heads, head_dim, seq));
    if (rc) return rc;
    return aeth_attn_kv8_launch(d_q, q_stride, d_layer, 0, nullptr, 0, 1, n, n_heads, kv_heads, head_dim, max_seq, seq, window, d_out,
                                d_ws, (hipStream_t)stream);
}

extern "C" AETH_API int aeth_attn_kv8_batch(const float* d_q, int64_t q_stride, const void* d_layers, int64_t layer_stride,
                                            const int32_t* d_lens, int64_t n_seqs, int64_t n_heads, int64_t kv_heads, int64_t head_dim,
                                            int64_t max_seq, int64_t max_len, int64_t window, float* d_out, void* d_ws,
                                            int64_t ws_bytes, void* stream) {
    const char* what = "aeth_attn_kv8_batch";
    if (!d_lens || ((uintptr_t)d_lens & 3) || max_len < 1) return aeth_set_error(AETH_EINVAL, "%s: bad argument (lengths)", what);
    int rc = aeth_attn_kv8_check(what, d_q, q_stride, d_layers, n_seqs, 1, n_heads, kv_heads, head_dim, max_seq, max_len, window, d_out, d_ws);
    if (!rc) rc = aeth_attn_kv8_check_ws(what, d_ws, ws_bytes, aeth_attn_kv8_ws(n_seqs, 1, n_heads, kv_heads, head_dim, max_len));
    if (!rc) rc = aeth_attn_kv8_check_slices(what, n_seqs, layer_stride, kv_heads, head_dim, max_seq);
    if (rc) return rc;
    return aeth_attn_kv8_launch(d_q, q_stride, d_layers, layer_stride, d_lens, 0, n_seqs, 1, n_heads, kv_heads, head_dim, max_seq, max_len,
                                window, d_out, d_ws, (hipStream_t)stream);
}
