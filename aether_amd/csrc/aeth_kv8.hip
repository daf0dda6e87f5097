// Writing an 8-bit key/value cache and reading it back (the layout: aeth_kv8.hpp),
// and the norm and rotation of queries and keys that stand before it.
//
// A token's K or V of one head, x of hd floats, is held as
//   scale s = fl32(amax / 127), codes c_i = 127·x_i / amax rounded to the nearest integer, ties to even,
// and stands for c_i · s. The quotient is rounded exactly, not the f32 quotient x_i / s, whose own
// rounding moves some codes next to a border: codes then do not depend on how they were computed.
// amax = 0 gives codes 0; a row with an infinity or NaN gets the scale NaN and codes 0, and every
// value of it reads back as NaN. The scale stands for one token and head: an append never touches
// what is there, and a prompt appended in pieces leaves the bytes of one appended whole.
#include <math.h>

#include <algorithm>

#include "aeth_common.hpp"
#include "aeth_internal.hpp"
#include "aeth_kv8.hpp"
#include "aeth_ops_internal.hpp"

typedef float kv8_f4 __attribute__((ext_vector_type(4)));

namespace {

// Rows read or written once, past the caches: 30000 tokens of 8 heads of 128 appended in 55 µs (72 with plain
// loads), read back in 48 (90 with plain stores, which displace the codes that a workgroup reads in pieces).
__device__ __forceinline__ float4 kv8_ld4(const float* p, bool vec) {
    if (vec) {
        const kv8_f4 v = __builtin_nontemporal_load((const kv8_f4*)p);
        return make_float4(v.x, v.y, v.z, v.w);
    }
    return make_float4(p[0], p[1], p[2], p[3]);
}

struct AppendArgs {
    uint8_t* cache;       // layer slice of the first sequence
    int64_t seq_bytes;    // from one sequence's slice to the next
    const int* slots;     // [seqs] the slot of each sequence's one token; nullptr: slot, n
    const float *k, *v;
    int64_t token_stride, head_stride;
    int64_t slot, n, max_seq;
    int nkv, tiles;       // tiles a head holds
    int vec;              // rows are 16-byte aligned
};

// Workgroup = (tile, KV head): 16 lanes a token, four rounds of 16 tokens. K codes go out from
// registers; V codes are transposed through LDS and go out 16 bytes at a time where the tile's tokens
// are all new, in words or bytes where some are not (those are left as they were). 30000 tokens of 8 heads of 128: 56 µs,
// 5.5 TB/s; 1999 of 64 from an odd slot 5.4 µs, 1.9 TB/s (256 workgroups, one wave of loads deep).
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_append(AppendArgs A) {
    constexpr int V4 = HD / 64, LW = HD / 4 + 4;  // float4s a lane and token; words of an LDS row
    __shared__ uint32_t vs[KV8_TILE * LW];
    const int h = blockIdx.x % A.nkv, tid = threadIdx.x, l16 = tid & 15, grp = tid >> 4;
    const int64_t slot = A.slot, n = A.n;
    const int64_t tile = (slot >> 6) + blockIdx.x / A.nkv;
    const int64_t first = tile * KV8_TILE - slot;  // the token at the tile's slot 0 (below 0: an older one)
    uint8_t* base = A.cache + ((int64_t)h * A.tiles + tile) * aeth_kv8_tile_bytes(HD);
    float4 x[4][2][V4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int64_t i = min(max(first + 16 * r + grp, (int64_t)0), n - 1);  // clamped: loaded, not stored
        const int64_t off = i * A.token_stride + h * A.head_stride + 4 * l16;
#pragma unroll
        for (int u = 0; u < V4; u++) {
            x[r][0][u] = kv8_ld4(A.k + off + 64 * u, A.vec);
            x[r][1][u] = kv8_ld4(A.v + off + 64 * u, A.vec);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int t = 16 * r + grp;
        const bool is_new = first + t >= 0 && first + t < n;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            uint32_t m = 0;
#pragma unroll
            for (int u = 0; u < V4; u++) m = kv8_abs_max(m, x[r][p][u]);
            m = kv8_umax<16>(m);
            const bool finite = m < 0x7F800000u;
            const float amax = __uint_as_float(m);
            const double inv = finite && m > 0 ? kv8_inverse(amax) : 0.0;
#pragma unroll
            for (int u = 0; u < V4; u++) {
                const uint32_t w = kv8_code4(x[r][p][u], inv, finite);
                if (p == 1) vs[t * LW + 16 * u + l16] = w;
                else if (is_new) *(uint32_t*)(base + t * HD + 64 * u + 4 * l16) = w;
            }
            if (is_new && l16 == 0)
                *(float*)(base + 2 * KV8_TILE * HD + 4 * (KV8_TILE * p + t)) = finite ? amax / 127.0f : __uint_as_float(0x7FC00000u);
        }
    }
    __syncthreads();
    // unit (four dimensions, token group g): 16 words of LDS, four rows of 16 bytes
    for (int unit = tid; unit < HD; unit += 256) {
        const int g = unit & 3, d4 = unit >> 2;
        uint32_t o[4][4];  // [dimension][word j]: tokens 16j + 4g + 0 .. 3
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t w[4], tr[4];
#pragma unroll
            for (int r = 0; r < 4; r++) w[r] = vs[(16 * j + 4 * g + r) * LW + d4];
            kv8_transpose4(w[0], w[1], w[2], w[3], tr);
#pragma unroll
            for (int d = 0; d < 4; d++) o[d][j] = tr[d];
        }
        uint8_t* dst = base + KV8_TILE * HD + 4 * d4 * KV8_TILE + 16 * g;
        if (first >= 0 && first + KV8_TILE <= n) {
#pragma unroll
            for (int d = 0; d < 4; d++) *(uint4*)(dst + d * KV8_TILE) = make_uint4(o[d][0], o[d][1], o[d][2], o[d][3]);
            continue;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t i0 = first + 16 * j + 4 * g;
            if (i0 >= 0 && i0 + 4 <= n) {
#pragma unroll
                for (int d = 0; d < 4; d++) *(uint32_t*)(dst + d * KV8_TILE + 4 * j) = o[d][j];
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (i0 + r >= 0 && i0 + r < n)
#pragma unroll
                        for (int d = 0; d < 4; d++) dst[d * KV8_TILE + 4 * j + r] = (uint8_t)(o[d][j] >> (8 * r));
            }
        }
    }
}

// Without a tile's staging, for a few tokens or one for each of many sequences: HD / 8 lanes a token, head and K or V; V's codes go out as bytes
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_append_few(AppendArgs A, int rows) {
    constexpr int L = HD / 8;
    const int unit = (blockIdx.x * 256 + threadIdx.x) / L, all = 2 * rows * A.nkv, u = min(unit, all - 1), e = 4 * (threadIdx.x % L);
    const int v = u & 1, h = (u >> 1) % A.nkv, row = (u >> 1) / A.nkv;
    const float* src = (v ? A.v : A.k) + row * A.token_stride + h * A.head_stride + e;
    const float4 a = kv8_ld4(src, A.vec), b = kv8_ld4(src + HD / 2, A.vec);
    const int64_t slot = A.slots ? (int64_t)A.slots[row] : A.slot + row;
    uint8_t* tiles = A.cache + (A.slots ? row : 0) * A.seq_bytes + (int64_t)h * A.tiles * aeth_kv8_tile_bytes(HD);
    const Kv8Row q = kv8_quantise<HD>(a, b);
    if (unit < all && slot >= 0 && slot < A.max_seq) kv8_put<HD>(tiles, slot, v, e, q);  // a full cache takes nothing
}

struct ReadArgs {
    const uint8_t* cache;
    float *k, *v;
    int64_t token_stride, head_stride, slot, n;
    int nkv, tiles, vec;
};

__device__ __forceinline__ void kv8_store4(float* p, uint32_t w, float s, bool vec) {
    const float4 y = make_float4((float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s, (float)(int8_t)(w >> 16) * s,
                                 (float)((int)w >> 24) * s);
    if (vec) __builtin_nontemporal_store((kv8_f4){y.x, y.y, y.z, y.w}, (kv8_f4*)p);
    else p[0] = y.x, p[1] = y.y, p[2] = y.z, p[3] = y.w;
}

// Workgroup = (tile, KV head): K a word a lane; V by units of four dimensions and eight tokens, four 8-byte
// pieces of its rows transposed in registers, so that a lane writes four dimensions of a token at once. 30000 tokens of
// 8 heads of 128: 48.5 µs, 6.4 TB/s; one token 3.5 µs (its tile's bytes, a launch).
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_read(ReadArgs A) {
    const int h = blockIdx.x % A.nkv, tid = threadIdx.x;
    const int64_t tile = (A.slot >> 6) + blockIdx.x / A.nkv;
    const int64_t first = tile * KV8_TILE - A.slot;
    const uint8_t* base = A.cache + ((int64_t)h * A.tiles + tile) * aeth_kv8_tile_bytes(HD);
    const float* sk = (const float*)(base + 2 * KV8_TILE * HD);
    const float* sv = sk + KV8_TILE;
    constexpr int KW = HD / 16;  // words of K a thread
    uint32_t kw[KW];
#pragma unroll
    for (int u = 0; u < KW; u++) kw[u] = *(const uint32_t*)(base + 4 * (tid + 256 * u));
    // V: unit (four dimensions, token group g, half of j)
    for (int unit = tid; unit < 2 * HD; unit += 256) {
        const int d4 = unit % (HD / 4), g = unit / (HD / 4) % 4, half = unit / HD;
        uint2 row[4];
#pragma unroll
        for (int d = 0; d < 4; d++) row[d] = *(const uint2*)(base + KV8_TILE * HD + (4 * d4 + d) * KV8_TILE + 16 * g + 8 * half);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            uint32_t w[4];
            if (j == 0) kv8_transpose4(row[0].x, row[1].x, row[2].x, row[3].x, w);
            else kv8_transpose4(row[0].y, row[1].y, row[2].y, row[3].y, w);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = 16 * (2 * half + j) + 4 * g + r;
                const int64_t i = first + t;
                if (i >= 0 && i < A.n) kv8_store4(A.v + i * A.token_stride + h * A.head_stride + 4 * d4, w[r], sv[t], A.vec);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < KW; u++) {
        const int at = tid + 256 * u, t = at / (HD / 4), d4 = at % (HD / 4);
        const int64_t i = first + t;
        if (i >= 0 && i < A.n) kv8_store4(A.k + i * A.token_stride + h * A.head_stride + 4 * d4, kw[u], sk[t], A.vec);
    }
}

int check_cache(const char* what, int64_t nkv, int64_t hd, int64_t max_seq) {
    if (nkv <= 0 || nkv > 65535 || max_seq <= 0 || max_seq > KV8_MAX_SEQ)
        return aeth_set_error(AETH_EINVAL, "%s: bad cache shape (kv_heads %lld, max_seq %lld)", what, (long long)nkv, (long long)max_seq);
    if (!aeth_kv8_head_dim(hd))
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: head_dim %lld (needs 64, 128 or 256)", what, (long long)hd);
    return AETH_OK;
}

// |(rows - 1)·token_stride + (heads - 1)·head_stride + hd| stays an int64 number of bytes, and rows do not overlap backwards
bool strides_ok(int64_t rows, int64_t nkv, int64_t hd, int64_t ts, int64_t hs) {
    int64_t a, b, c;
    return ts >= 0 && hs >= 0 && (rows == 1 || ts >= hd) && (nkv == 1 || hs >= hd) && aeth_mul_ok(rows, ts, &a) &&
           aeth_mul_ok(nkv, hs, &b) && !__builtin_add_overflow(a, b, &c) && c < INT64_MAX / 8;
}

bool aligned16(const void* a, const void* b, int64_t ts, int64_t hs) {
    return ((((uintptr_t)a | (uintptr_t)b) & 15) == 0) && ((ts | hs) & 3) == 0;
}

}  // namespace

// Tokens whose rows go a 16th of a wave each rather than by tiles: while rows times heads leave the chip half idle. 8 heads of
// 128: 1 token 2.4 µs against 4.3, 256 tokens 3.9 and 5.1, 512 tokens 5.5 and 5.2, 1000 tokens 8.8 and 5.2.
static bool append_few(int64_t rows, int64_t nkv) { return rows < 14 * (int64_t)aeth_num_cus() / nkv; }

int aeth_kv8_append_launch(void* cache, int64_t seq_bytes, const int* d_slots, int64_t seqs, const float* k, const float* v,
                           int64_t token_stride, int64_t head_stride, int64_t n, int64_t nkv, int64_t hd, int64_t max_seq,
                           int64_t slot, hipStream_t s) {
    if (n <= 0 || seqs <= 0) return AETH_OK;
    AppendArgs A;
    A.cache = (uint8_t*)cache;
    A.seq_bytes = seq_bytes;
    A.slots = d_slots;
    A.k = k;
    A.v = v;
    A.token_stride = token_stride;
    A.head_stride = head_stride;
    A.slot = slot;
    A.n = n;
    A.max_seq = max_seq;
    A.nkv = (int)nkv;
    A.tiles = (int)aeth_cdiv(max_seq, KV8_TILE);
    A.vec = aligned16(k, v, token_stride, head_stride);
    const dim3 block(256);
    const int64_t rows = d_slots ? seqs : n;
    if (d_slots || append_few(n, nkv)) {
        const dim3 grid((unsigned)aeth_cdiv(2 * rows * nkv * (hd / 8), 256));
        if (hd == 64) hipLaunchKernelGGL(k_kv8_append_few<64>, grid, block, 0, s, A, (int)rows);
        else if (hd == 128) hipLaunchKernelGGL(k_kv8_append_few<128>, grid, block, 0, s, A, (int)rows);
        else hipLaunchKernelGGL(k_kv8_append_few<256>, grid, block, 0, s, A, (int)rows);
        AETH_LAUNCH_CHECK();
        return AETH_OK;
    }
    const dim3 grid((unsigned)((((slot + n - 1) >> 6) - (slot >> 6) + 1) * nkv));
    if (hd == 64) hipLaunchKernelGGL(k_kv8_append<64>, grid, block, 0, s, A);
    else if (hd == 128) hipLaunchKernelGGL(k_kv8_append<128>, grid, block, 0, s, A);
    else hipLaunchKernelGGL(k_kv8_append<256>, grid, block, 0, s, A);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

int aeth_kv8_read_launch(const void* cache, float* k, float* v, int64_t token_stride, int64_t head_stride, int64_t n,
                         int64_t nkv, int64_t hd, int64_t max_seq, int64_t slot, hipStream_t s) {
    if (n <= 0) return AETH_OK;
    ReadArgs A;
    A.cache = (const uint8_t*)cache;
    A.k = k;
    A.v = v;
    A.token_stride = token_stride;
    A.head_stride = head_stride;
    A.slot = slot;
    A.n = n;
    A.nkv = (int)nkv;
    A.tiles = (int)aeth_cdiv(max_seq, KV8_TILE);
    A.vec = aligned16(k, v, token_stride, head_stride);
    const dim3 grid((unsigned)((((slot + n - 1) >> 6) - (slot >> 6) + 1) * nkv)), block(256);
    if (hd == 64) hipLaunchKernelGGL(k_kv8_read<64>, grid, block, 0, s, A);
    else if (hd == 128) hipLaunchKernelGGL(k_kv8_read<128>, grid, block, 0, s, A);
    else hipLaunchKernelGGL(k_kv8_read<256>, grid, block, 0, s, A);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

extern "C" AETH_API int64_t aeth_kv8_layer_bytes(int64_t kv_heads, int64_t head_dim, int64_t max_seq) {
    if (check_cache("aeth_kv8_layer_bytes", kv_heads, head_dim, max_seq)) return -1;
    return kv_heads * aeth_cdiv(max_seq, KV8_TILE) * aeth_kv8_tile_bytes((int)head_dim);
}

// what a call on n tokens from `slot` of one sequence has to be
static int check_range(const char* what, const void* cache, const void* k, const void* v, int64_t ts, int64_t hs, int64_t n,
                       int64_t nkv, int64_t hd, int64_t max_seq, int64_t slot) {
    if (!cache || !k || !v || ((uintptr_t)cache & 15) || (((uintptr_t)k | (uintptr_t)v) & 3))
        return aeth_set_error(AETH_EINVAL, "%s: bad argument (the cache 16-byte aligned, rows 4-byte)", what);
    int rc = check_cache(what, nkv, hd, max_seq);
    if (rc) return rc;
    if (n < 0 || slot < 0 || slot > max_seq || n > max_seq - slot)
        return aeth_set_error(AETH_EINVAL, "%s: %lld tokens from slot %lld of %lld", what, (long long)n, (long long)slot, (long long)max_seq);
    if (!strides_ok(n, nkv, hd, ts, hs))
        return aeth_set_error(AETH_EINVAL, "%s: strides %lld / %lld of rows of %lld", what, (long long)ts, (long long)hs, (long long)hd);
    if (aeth_cdiv(n, KV8_TILE) * nkv > (int64_t)1 << 23)  // workgroups of 256 threads within the grid's 2^32
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld tokens of %lld heads in one call", what, (long long)n, (long long)nkv);
    return AETH_OK;
}

extern "C" AETH_API int aeth_kv8_append(void* d_layer, const float* d_k, const float* d_v, int64_t token_stride,
                                        int64_t head_stride, int64_t n, int64_t kv_heads, int64_t head_dim, int64_t max_seq,
                                        int64_t slot, void* stream) {
    const int rc = check_range("aeth_kv8_append", d_layer, d_k, d_v, token_stride, head_stride, n, kv_heads, head_dim, max_seq, slot);
    if (rc) return rc;
    return aeth_kv8_append_launch(d_layer, 0, nullptr, 1, d_k, d_v, token_stride, head_stride, n, kv_heads, head_dim, max_seq,
                                  slot, (hipStream_t)stream);
}

extern "C" AETH_API int aeth_kv8_append_batch(void* d_layers, int64_t layer_stride, const int32_t* d_slots, const float* d_k,
                                              const float* d_v, int64_t token_stride, int64_t head_stride, int64_t n_seqs,
                                              int64_t kv_heads, int64_t head_dim, int64_t max_seq, void* stream) {
    const char* what = "aeth_kv8_append_batch";
    if (!d_layers || !d_slots || !d_k || !d_v || ((uintptr_t)d_layers & 15) || (layer_stride & 15) ||
        (((uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_slots) & 3))
        return aeth_set_error(AETH_EINVAL, "%s: bad argument (slices 16-byte aligned, rows 4-byte)", what);
    int rc = check_cache(what, kv_heads, head_dim, max_seq);
    if (rc) return rc;
    int64_t all;
    if (n_seqs < 0 || n_seqs > 65535 || (n_seqs > 1 && layer_stride < aeth_kv8_layer_bytes(kv_heads, head_dim, max_seq)) ||
        layer_stride < 0 || !aeth_mul_ok(n_seqs, layer_stride, &all))
        return aeth_set_error(AETH_EINVAL, "%s: %lld sequences %lld bytes apart", what, (long long)n_seqs, (long long)layer_stride);
    if (!strides_ok(n_seqs, kv_heads, head_dim, token_stride, head_stride))
        return aeth_set_error(AETH_EINVAL, "%s: strides %lld / %lld of rows of %lld", what, (long long)token_stride,
                              (long long)head_stride, (long long)head_dim);
    if (n_seqs * kv_heads > (int64_t)1 << 25)  // 2·hd/8 threads each within the grid's 2^32
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld sequences of %lld heads in one call", what, (long long)n_seqs, (long long)kv_heads);
    return aeth_kv8_append_launch(d_layers, layer_stride, d_slots, n_seqs, d_k, d_v, token_stride, head_stride, 1, kv_heads,
                                  head_dim, max_seq, 0, (hipStream_t)stream);
}

extern "C" AETH_API int aeth_kv8_read(const void* d_layer, float* d_k, float* d_v, int64_t token_stride, int64_t head_stride,
                                      int64_t n, int64_t kv_heads, int64_t head_dim, int64_t max_seq, int64_t slot,
                                      void* stream) {
    const int rc = check_range("aeth_kv8_read", d_layer, d_k, d_v, token_stride, head_stride, n, kv_heads, head_dim, max_seq, slot);
    if (rc) return rc;
    return aeth_kv8_read_launch(d_layer, d_k, d_v, token_stride, head_stride, n, kv_heads, head_dim, max_seq, slot, (hipStream_t)stream);
}

// ── norm and rotation of queries and keys ─────────────────────────────────
// Head h of a row: y = x / sqrt(Σx²/hd + eps) · w (w the queries' or the keys' weight; neither: y = x), then the
// rotation of the halves (y_i, y_{i+hd/2}) by the table row min(pos, max_seq - 1), as aeth_rmsnorm and aeth_rope do.
namespace {
struct QkArgs {
    const float* x;
    int64_t x_stride;
    float* out;
    int64_t out_stride;
    const float *qw, *kw;  // nullptr: no norm of those heads
    float eps;
    int64_t pos;
    const int* d_pos;      // [n] instead of pos + i
    const float *sin_t, *cos_t;
    int64_t n, max_seq;
    int nq, heads, hd;     // query heads; query and key heads
};

constexpr int QK_MAX_HD = 512, QK_MAX_AXES = 16;  // with several axes: the pairs' axes go as a kernel argument
struct QkAxes {
    int64_t pos_stride;                   // d_pos is [axes][pos_stride]
    uint32_t axis[QK_MAX_HD / 2 / 4];     // the axis of each pair, a byte each
};

__device__ __forceinline__ int64_t qk_row(const QkArgs& A, int64_t i) {
    const int64_t p = A.d_pos ? (int64_t)A.d_pos[i] : A.pos + i;
    return min(max(p, (int64_t)0), A.max_seq - 1);
}
__device__ __forceinline__ int64_t qk_row(const QkArgs& A, const QkAxes& X, int64_t i, int axis) {
    return min(max((int64_t)A.d_pos[axis * X.pos_stride + i], (int64_t)0), A.max_seq - 1);
}

// sum over aligned groups of L lanes (8, 16 or 32), the same value in each
template <int L>
__device__ __forceinline__ float qk_sum(float v) {
    v += aeth_dpp_xor1f(v);
    v += aeth_dpp_xor2f(v);
    v += aeth_dpp_mirror8f(v);
    if (L >= 16) v += aeth_dpp_mirror16f(v);
    if (L >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return v;
}

// hd / 8 lanes a head, four pairs a lane; rows, weights and tables 16-byte aligned
template <int HD>
__global__ void __launch_bounds__(256) k_qk_norm_rope_v(QkArgs A) {
    constexpr int L = HD / 8, HALF = HD / 2;
    const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / L, all = (uint32_t)A.n * A.heads;  // at most 2^25 units
    const uint32_t u = min(unit, all - 1), row = u / (uint32_t)A.heads;  // past the end: loaded, not stored (whole waves stay active)
    const int64_t i = row;
    const int h = (int)(u - row * A.heads), e = 4 * (threadIdx.x % L);
    const float* src = A.x + i * A.x_stride + (int64_t)h * HD + e;
    float4 a = *(const float4*)src, b = *(const float4*)(src + HALF);
    const int64_t p = qk_row(A, i);
    const float4 sn = *(const float4*)(A.sin_t + p * HALF + e), cs = *(const float4*)(A.cos_t + p * HALF + e);
    const float* w = h < A.nq ? A.qw : A.kw;
    if (A.qw || A.kw) {  // (uniform)
        const float4 wa = w ? *(const float4*)(w + e) : make_float4(1, 1, 1, 1), wb = w ? *(const float4*)(w + e + HALF) : wa;
        const float ss = qk_sum<L>(((a.x * a.x + a.y * a.y) + (a.z * a.z + a.w * a.w)) + ((b.x * b.x + b.y * b.y) + (b.z * b.z + b.w * b.w)));
        const float rms = w ? sqrtf(ss / (float)HD + A.eps) : 1.0f;
        a = make_float4(a.x / rms * wa.x, a.y / rms * wa.y, a.z / rms * wa.z, a.w / rms * wa.w);
        b = make_float4(b.x / rms * wb.x, b.y / rms * wb.y, b.z / rms * wb.z, b.w / rms * wb.w);
    }
    if (unit >= all) return;
    float* dst = A.out + i * A.out_stride + (int64_t)h * HD + e;
    kv8_rotate(a, b, sn, cs);
    // streaming stores: 4000 rows of 32 + 8 heads of 128 in 25.1 µs (6.6 TB/s) against 27.4
    __builtin_nontemporal_store((kv8_f4){a.x, a.y, a.z, a.w}, (kv8_f4*)dst);
    __builtin_nontemporal_store((kv8_f4){b.x, b.y, b.z, b.w}, (kv8_f4*)(dst + HALF));
}

// Σx² of four, rounded as it is in k_qk_norm_rope_v: where the axes agree both give the same bits
__device__ __forceinline__ float qk_squares(float4 a) { return fmaf(a.x, a.x, a.y * a.y) + fmaf(a.z, a.z, a.w * a.w); }

// Several axes: the four pairs of a lane take their table entries one by one, each from the row of its axis' position, and
// serve HEADS heads of the token: four, where that leaves each CU four workgroups, else one. 4000 rows of 32 + 8 heads of 128 by three axes 27 µs
// (6.1 TB/s; with inputs not in the caches 34); one head a thread 50, two, three, eight in turn 38, 36, 39 against those 34.
template <int HD, int HEADS>
__global__ void __launch_bounds__(256) k_qk_norm_rope_axes_v(QkArgs A, QkAxes X) {
    constexpr int L = HD / 8, HALF = HD / 2;
    const uint32_t groups = ((uint32_t)A.heads + HEADS - 1) / HEADS;  // of a row
    const uint32_t unit = (blockIdx.x * 256u + threadIdx.x) / L, all = (uint32_t)A.n * groups;  // at most 2^25 units
    const uint32_t u = min(unit, all - 1), row = u / groups;  // past the end: loaded, not stored (whole waves stay active)
    const int64_t i = row;
    const int h0 = (int)(u - row * groups) * HEADS, e = 4 * (threadIdx.x % L);
    const float* src = A.x + i * A.x_stride + e;
    float4 a[HEADS], b[HEADS];
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
        const float* p = src + (int64_t)min(h0 + j, A.heads - 1) * HD;
        a[j] = *(const float4*)p;
        b[j] = *(const float4*)(p + HALF);
    }
    const uint32_t axes = X.axis[e / 4];
    int64_t at[4];
#pragma unroll
    for (int j = 0; j < 4; j++) at[j] = qk_row(A, X, i, axes >> (8 * j) & 0xFFu) * HALF + e + j;
    const float4 sn = make_float4(A.sin_t[at[0]], A.sin_t[at[1]], A.sin_t[at[2]], A.sin_t[at[3]]);
    const float4 cs = make_float4(A.cos_t[at[0]], A.cos_t[at[1]], A.cos_t[at[2]], A.cos_t[at[3]]);
    // the weights of the first head's kind, which nearly always serve the others too
    const float* w0 = h0 < A.nq ? A.qw : A.kw;
    const float4 one = make_float4(1, 1, 1, 1), wa0 = w0 ? *(const float4*)(w0 + e) : one, wb0 = w0 ? *(const float4*)(w0 + e + HALF) : one;
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
        const int h = min(h0 + j, A.heads - 1);
        if (A.qw || A.kw) {  // (uniform)
            const float* w = w0;
            float4 wa = wa0, wb = wb0;
            if (h0 < A.nq && h >= A.nq) {
                w = A.kw;
                wa = w ? *(const float4*)(w + e) : one;
                wb = w ? *(const float4*)(w + e + HALF) : one;
            }
            const float ss = qk_sum<L>(qk_squares(a[j]) + qk_squares(b[j]));
            const float rms = w ? sqrtf(ss / (float)HD + A.eps) : 1.0f;
            a[j] = make_float4(a[j].x / rms * wa.x, a[j].y / rms * wa.y, a[j].z / rms * wa.z, a[j].w / rms * wa.w);
            b[j] = make_float4(b[j].x / rms * wb.x, b[j].y / rms * wb.y, b[j].z / rms * wb.z, b[j].w / rms * wb.w);
        }
        kv8_rotate(a[j], b[j], sn, cs);
        if (unit >= all || h0 + j >= A.heads) continue;
        float* dst = A.out + i * A.out_stride + (int64_t)h * HD + e;
        __builtin_nontemporal_store((kv8_f4){a[j].x, a[j].y, a[j].z, a[j].w}, (kv8_f4*)dst);
        __builtin_nontemporal_store((kv8_f4){b[j].x, b[j].y, b[j].z, b[j].w}, (kv8_f4*)(dst + HALF));
    }
}

// any even hd, any alignment: a wave a head, lanes over the pairs (read again for the rotation: the row is in cache)
template <bool AXES>
__device__ __forceinline__ void qk_norm_rope(const QkArgs& A, const QkAxes& X) {
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (unit >= A.n * A.heads) return;
    const int64_t i = unit / A.heads;
    const int h = (int)(unit % A.heads), lane = threadIdx.x & 63, half = A.hd / 2;
    const float* src = A.x + i * A.x_stride + (int64_t)h * A.hd;
    float* dst = A.out + i * A.out_stride + (int64_t)h * A.hd;
    const int64_t p = AXES ? 0 : qk_row(A, i);
    const float* w = h < A.nq ? A.qw : A.kw;
    float rms = 1.0f;
    if (w) {
        float ss = 0.0f;
        for (int e = lane; e < A.hd; e += 64) ss += src[e] * src[e];
        rms = sqrtf(aeth_wave_sum(ss) / (float)A.hd + A.eps);
    }
    for (int e = lane; e < half; e += 64) {
        const int64_t at = (AXES ? qk_row(A, X, i, X.axis[e >> 2] >> (8 * (e & 3)) & 0xFFu) : p) * half + e;
        const float sn = A.sin_t[at], cs = A.cos_t[at];
        float a = src[e], b = src[e + half];
        if (w) {
            a = a / rms * w[e];
            b = b / rms * w[e + half];
        }
        dst[e] = kv8_rot0(a, b, sn, cs);
        dst[e + half] = kv8_rot1(a, b, sn, cs);
    }
}
__global__ void __launch_bounds__(256) k_qk_norm_rope(QkArgs A) { qk_norm_rope<false>(A, {}); }
__global__ void __launch_bounds__(256) k_qk_norm_rope_axes(QkArgs A, QkAxes X) { qk_norm_rope<true>(A, X); }
}  // namespace

template <int HD>
static void qk_launch_axes(const QkArgs& A, const QkAxes& X, hipStream_t s) {
    auto grid = [&](int64_t heads) { return dim3((unsigned)aeth_cdiv(A.n * aeth_cdiv(A.heads, heads) * (HD / 8), 256)); };
    if (grid(4).x >= 4u * (unsigned)aeth_num_cus()) hipLaunchKernelGGL((k_qk_norm_rope_axes_v<HD, 4>), grid(4), dim3(256), 0, s, A, X);
    else hipLaunchKernelGGL((k_qk_norm_rope_axes_v<HD, 1>), grid(1), dim3(256), 0, s, A, X);
}

// X: several axes (nullptr: one)
static int qk_launch(const QkArgs& A, const QkAxes* X, hipStream_t s) {
    if (A.n <= 0 || A.heads <= 0) return AETH_OK;
    const bool al16 = ((((uintptr_t)A.x | (uintptr_t)A.out | (uintptr_t)A.qw | (uintptr_t)A.kw | (uintptr_t)A.sin_t | (uintptr_t)A.cos_t) & 15) == 0) &&
                      ((A.x_stride | A.out_stride) & 3) == 0;
    const int hd = A.hd;
    const dim3 block(256);
    if (al16 && (hd == 64 || hd == 128 || hd == 256)) {
        const dim3 grid((unsigned)aeth_cdiv(A.n * A.heads * (hd / 8), 256));
        if (X) {
            if (hd == 64) qk_launch_axes<64>(A, *X, s);
            else if (hd == 128) qk_launch_axes<128>(A, *X, s);
            else qk_launch_axes<256>(A, *X, s);
        } else {
            if (hd == 64) hipLaunchKernelGGL(k_qk_norm_rope_v<64>, grid, block, 0, s, A);
            else if (hd == 128) hipLaunchKernelGGL(k_qk_norm_rope_v<128>, grid, block, 0, s, A);
            else hipLaunchKernelGGL(k_qk_norm_rope_v<256>, grid, block, 0, s, A);
        }
    } else {
        const dim3 grid((unsigned)aeth_cdiv(A.n * A.heads, 4));
        if (X) hipLaunchKernelGGL(k_qk_norm_rope_axes, grid, block, 0, s, A, *X);
        else hipLaunchKernelGGL(k_qk_norm_rope, grid, block, 0, s, A);
    }
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

int aeth_qk_norm_rope_launch(const float* x, int64_t x_stride, int64_t n, int64_t n_heads, int64_t kv_heads, int64_t hd,
                             const float* qw, const float* kw, float eps, int64_t pos, const int* d_pos, const float* sin_t,
                             const float* cos_t, int64_t max_seq, float* out, int64_t out_stride, hipStream_t s) {
    const int64_t heads = n_heads + kv_heads;
    if (n <= 0 || heads <= 0) return AETH_OK;
    const QkArgs A{x, x_stride, out, out_stride, qw, kw, eps, pos, d_pos, sin_t, cos_t, n, max_seq, (int)n_heads, (int)heads, (int)hd};
    return qk_launch(A, nullptr, s);
}

// what the two entry points ask of their arguments in common
static int check_qk(const char* what, const float* d_x, int64_t x_stride, int64_t n, int64_t n_heads, int64_t kv_heads, int64_t head_dim,
                    const float* d_sin, const float* d_cos, int64_t max_seq, const float* d_out, int64_t out_stride) {
    if (!d_x || !d_sin || !d_cos || !d_out || n < 0 || n_heads < 0 || kv_heads < 0 || max_seq <= 0 || head_dim <= 0 || head_dim % 2)
        return aeth_set_error(AETH_EINVAL, "%s: bad argument", what);
    if (n_heads > 65535 || kv_heads > 65535 || head_dim > 65536)
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld + %lld heads of %lld", what, (long long)n_heads, (long long)kv_heads, (long long)head_dim);
    const int64_t row = (n_heads + kv_heads) * head_dim;
    int64_t a, b;
    if (x_stride < row || out_stride < row || !aeth_mul_ok(n, x_stride, &a) || !aeth_mul_ok(n, out_stride, &b) ||
        a > INT64_MAX / 4 || b > INT64_MAX / 4)
        return aeth_set_error(AETH_EINVAL, "%s: strides %lld / %lld of rows of %lld", what, (long long)x_stride, (long long)out_stride, (long long)row);
    if (d_out == d_x && x_stride != out_stride && n > 1)
        return aeth_set_error(AETH_EINVAL, "%s: in place with another row stride", what);
    if (n * (n_heads + kv_heads) > (int64_t)1 << 25)  // workgroups of 256 threads within the grid's 2^32
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld rows of %lld heads in one call", what, (long long)n, (long long)(n_heads + kv_heads));
    return AETH_OK;
}

extern "C" AETH_API int aeth_qk_norm_rope(const float* d_x, int64_t x_stride, int64_t n, int64_t n_heads, int64_t kv_heads,
                                          int64_t head_dim, const float* d_qw, const float* d_kw, float eps, int64_t pos,
                                          const int32_t* d_pos, const float* d_sin, const float* d_cos, int64_t max_seq,
                                          float* d_out, int64_t out_stride, void* stream) {
    const char* what = "aeth_qk_norm_rope";
    if (pos < 0 || pos > INT64_MAX - std::max<int64_t>(n, 0)) return aeth_set_error(AETH_EINVAL, "%s: bad argument", what);
    const int rc = check_qk(what, d_x, x_stride, n, n_heads, kv_heads, head_dim, d_sin, d_cos, max_seq, d_out, out_stride);
    if (rc) return rc;
    return aeth_qk_norm_rope_launch(d_x, x_stride, n, n_heads, kv_heads, head_dim, d_qw, d_kw, eps, pos, d_pos, d_sin, d_cos, max_seq,
                                    d_out, out_stride, (hipStream_t)stream);
}

extern "C" AETH_API int aeth_qk_norm_rope_axes(const float* d_x, int64_t x_stride, int64_t n, int64_t n_heads, int64_t kv_heads,
                                               int64_t head_dim, const float* d_qw, const float* d_kw, float eps, const int32_t* d_pos,
                                               int64_t pos_stride, int64_t n_axes, const int32_t* pair_axes, const float* d_sin,
                                               const float* d_cos, int64_t max_seq, float* d_out, int64_t out_stride, void* stream) {
    const char* what = "aeth_qk_norm_rope_axes";
    if (!d_pos || ((uintptr_t)d_pos & 3) || !pair_axes) return aeth_set_error(AETH_EINVAL, "%s: bad argument (positions, axes)", what);
    const int rc = check_qk(what, d_x, x_stride, n, n_heads, kv_heads, head_dim, d_sin, d_cos, max_seq, d_out, out_stride);
    if (rc) return rc;
    if (head_dim > QK_MAX_HD || n_axes > QK_MAX_AXES)
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: heads of %lld turned by %lld axes (at most %d and %d)", what, (long long)head_dim,
                              (long long)n_axes, QK_MAX_HD, QK_MAX_AXES);
    int64_t all;
    if (n_axes < 1 || (n_axes > 1 && pos_stride < n) || pos_stride < 0 || !aeth_mul_ok(n_axes, pos_stride, &all) || all > INT64_MAX / 4)
        return aeth_set_error(AETH_EINVAL, "%s: %lld axes of positions %lld apart, of %lld rows", what, (long long)n_axes, (long long)pos_stride, (long long)n);
    QkAxes X = {};
    X.pos_stride = pos_stride;
    for (int64_t j = 0; j < head_dim / 2; j++) {
        if (pair_axes[j] < 0 || pair_axes[j] >= n_axes)
            return aeth_set_error(AETH_EINVAL, "%s: pair %lld of axis %d of %lld", what, (long long)j, (int)pair_axes[j], (long long)n_axes);
        X.axis[j / 4] |= (uint32_t)pair_axes[j] << (8 * (j % 4));
    }
    const QkArgs A{d_x, x_stride, d_out, out_stride, d_qw, d_kw, eps, 0, d_pos, d_sin, d_cos, n, max_seq, (int)n_heads, (int)(n_heads + kv_heads), (int)head_dim};
    return qk_launch(A, &X, (hipStream_t)stream);
}
