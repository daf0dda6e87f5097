// Eviction from the 8-bit cache (aeth_kv8.hpp) by the weight that each token has received.
//
// Of a head's len tokens `keep` stay: the first `first`, the last `recent`, and of the others the
// keep - first - recent of largest weight, the lower slot before the higher where weights are equal
// (NaN is below every number, -0 equals 0). They keep their order, their codes and their scales: a kept
// token stands for the same values as before. Three steps: the list of kept slots by head (k_kv8_select),
// the tokens gathered into the destination's tiles (k_kv8_gather), and, where the destination is the source, into
// tiles of the workspace and from there back (k_kv8_put_back): a tile may then be read by many workgroups
// before another has written it, with no order between them.
#include <math.h>

#include <algorithm>

#include "aeth_common.hpp"
#include "aeth_internal.hpp"
#include "aeth_kv8.hpp"
#include "aeth_ops_internal.hpp"

namespace {

struct EvictArgs {
    const uint8_t* cache;  // slice of the first sequence
    int64_t seq_bytes;
    const float* weights;  // [seqs][nkv][max_seq]
    const int* lens;       // [seqs], clamped to [0, max_len]; nullptr: max_len
    int64_t max_seq, max_len, keep, first, recent;
    int nkv, tiles;        // tiles a head's slice holds
    uint8_t* dst;
    int64_t dst_seq_bytes, dst_seq;
    int dst_tiles;
    float* dst_weights;    // [seqs][nkv][dst_seq]; nullptr: not moved
    int* dst_lens;         // [seqs]; nullptr: not written
    // between the steps: tokens kept [seqs][nkv]; their slots and weights [seqs][nkv][keep]
    int* rows;
    int* list;
    int64_t list_stride;
    float* kept_weights;
    int64_t most;          // min(keep, max_len)
    int gather_blocks;     // of a head; the blocks behind them write the weights
    int in_place;
};

__device__ __forceinline__ int64_t ev_len(const EvictArgs& A, int seq) {
    return A.lens ? min(max((int64_t)A.lens[seq], (int64_t)0), A.max_len) : A.max_len;
}

// weights as whole numbers in their order
__device__ __forceinline__ uint32_t ev_key(float w) {
    uint32_t f = __float_as_uint(w);
    f = f == 0x80000000u ? 0 : f;
    if ((f & 0x7FFFFFFFu) > 0x7F800000u) return 0;
    return f & 0x80000000u ? ~f : f | 0x80000000u;
}

constexpr int SEL = 1024;  // threads of a selection

// exclusive prefix sums of two counts below 2^16 each over the workgroup, packed in one word, and their totals
__device__ __forceinline__ uint32_t ev_scan(uint32_t v, uint32_t (*part)[SEL / 64], int round, uint32_t& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(x, d, 64);
        x += lane >= d ? y : 0;
    }
    if (lane == 63) part[round & 1][w] = x;
    __syncthreads();  // (the other buffer's readers have passed the barrier before this one)
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < SEL / 64; i++) {
        const uint32_t y = part[round & 1][i];
        before += i < w ? y : 0;
        total += y;
    }
    return before + x - v;
}

// One workgroup a head: the key of the last token chosen by three passes over its bits (11, 11, 10) with counts in LDS,
// then one pass that numbers the kept slots in order.
__global__ void __launch_bounds__(SEL) k_kv8_select(EvictArgs A) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t part[2][SEL / 64];
    __shared__ uint32_t found[2];
    const int tid = threadIdx.x, h = blockIdx.x, seq = blockIdx.y;
    const int64_t len = ev_len(A, seq), unit = (int64_t)seq * A.nkv + h;
    const float* w = A.weights + unit * A.max_seq;
    int* list = A.list + unit * A.list_stride;
    float* kw = A.kept_weights + unit * A.most;
    const int64_t rows = min(len, A.keep);
    if (tid == 0) A.rows[unit] = (int)rows;
    if (len <= A.keep) {  // (uniform) all stay
        for (int64_t t = tid; t < len; t += SEL) {
            list[t] = (int)t;
            kw[t] = w[t];
        }
        return;
    }
    const int64_t lo = A.first, hi = len - A.recent;  // the slots to choose from
    uint32_t need = (uint32_t)(A.keep - A.first - A.recent), prefix = 0;
    if (need > 0) {  // (uniform)
        int done = 0;
        for (int pass = 0; pass < 3; pass++) {
            const int bits = pass < 2 ? 11 : 10, shift = 32 - done - bits;
            for (int i = tid; i < 2048; i += SEL) hist[i] = 0;
            __syncthreads();
            for (int64_t t = lo + tid; t < hi; t += SEL) {
                const uint32_t k = ev_key(w[t]);
                if (done == 0 || k >> (32 - done) == prefix) atomicAdd(&hist[k >> shift & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            // the bin in which the need-th from the top lies: counts above each pair of bins
            const int b = 2046 - 2 * tid;  // thread 0: the highest two
            const uint32_t c1 = hist[b + 1], c0 = hist[b];
            // counts may pass 2^16: a scan of whole words
            uint32_t x = c0 + c1;
            const int lane = tid & 63, wv = tid >> 6;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t y = __shfl_up(x, d, 64);
                x += lane >= d ? y : 0;
            }
            if (lane == 63) part[0][wv] = x;
            __syncthreads();
            uint32_t above = x - c0 - c1;
            for (int i = 0; i < wv; i++) above += part[0][i];
            if (above < need && need <= above + c1) {
                found[0] = b + 1;
                found[1] = above;
            } else if (above + c1 < need && need <= above + c1 + c0) {
                found[0] = b;
                found[1] = above + c1;
            }
            __syncthreads();
            prefix = prefix << bits | found[0];
            need -= found[1];
            done += bits;
            __syncthreads();
        }
    }
    // prefix: the key of the last one chosen; `need` of its equals, from the lowest slot on. need 0 from the start: none
    const bool some = A.keep > A.first + A.recent;
    uint32_t equals = 0;
    int64_t at = 0;  // equal keys passed and slots listed so far
    int round = 0;
    for (int64_t t0 = 0; t0 < len; t0 += 4 * SEL, round++) {
        uint32_t key[4];
        float wt[4];
        bool sure[4], equal[4];
        uint32_t n_eq = 0, n_sure = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t t = t0 + 4 * tid + j;
            wt[j] = t < len ? w[t] : 0.0f;
            key[j] = ev_key(wt[j]);
            const bool ends = t < len && (t < lo || t >= hi), mid = t >= lo && t < hi;
            sure[j] = ends || (mid && some && key[j] > prefix);
            equal[j] = mid && some && key[j] == prefix;
            n_eq += equal[j];
            n_sure += sure[j];
        }
        uint32_t total;
        const uint32_t before = ev_scan(n_sure << 16 | n_eq, part, round, total);
        // equals taken before a slot: those passed, up to `need`
        uint32_t eq = equals + (before & 0xFFFFu);
        int64_t pos = at + (before >> 16) + min(eq, need) - min(equals, need);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const bool take = sure[j] || (equal[j] && eq < need);
            eq += equal[j];
            if (take) {
                list[pos] = (int)(t0 + 4 * tid + j);
                kw[pos] = wt[j];
                pos++;
            }
        }
        const uint32_t all = equals + (total & 0xFFFFu);
        at += (total >> 16) + min(all, need) - min(equals, need);
        equals = all;
    }
}

// A tile's bytes from `src`, the same tile elsewhere, or token by token through `from` (LDS: the source slot of each token);
// tokens behind the first n keep what is there.
template <int HD>
__device__ __forceinline__ void ev_tile(uint8_t* dst, const uint8_t* head, const int* from, int n) {
    const int tid = threadIdx.x;
    constexpr int64_t TB = aeth_kv8_tile_bytes(HD);
#pragma unroll
    for (int u = 0; u < HD / 64; u++) {  // K: pieces of 16 bytes
        const int at = tid + 256 * u, t = at / (HD / 16), e = 16 * (at % (HD / 16));
        if (t < n) {
            const int s = from[t];
            *(uint4*)(dst + t * HD + e) = *(const uint4*)(head + (s >> 6) * TB + (s & 63) * HD + e);
        }
    }
    {   // V: a thread takes the four tokens of a word of a row, every 16th row
        const int word = tid & 15, t = 16 * (word & 3) + 4 * (word >> 2);
        const uint8_t* src[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int s = from[min(t + j, n - 1)];
            src[j] = head + (s >> 6) * TB + KV8_TILE * HD + aeth_kv8_vbyte(s & 63);
        }
        uint8_t* out = dst + KV8_TILE * HD + 4 * word;
#pragma unroll 4
        for (int d = tid >> 4; d < HD; d += 16) {
            uint32_t b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) b[j] = src[j][d * KV8_TILE];
            if (t + 3 < n) *(uint32_t*)(out + d * KV8_TILE) = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
            else {
#pragma unroll
                for (int j = 0; j < 3; j++)
                    if (t + j < n) out[d * KV8_TILE + j] = (uint8_t)b[j];
            }
        }
    }
    if (tid < 2 * KV8_TILE) {
        const int t = tid & 63, v = tid >> 6;
        if (t < n) {
            const int s = from[t];
            *(float*)(dst + 2 * KV8_TILE * HD + 4 * tid) = *(const float*)(head + (s >> 6) * TB + 2 * KV8_TILE * HD + 4 * (KV8_TILE * v + (s & 63)));
        }
    }
}

// The kept tokens' weights at the front of a head's row, zeros behind them
__device__ __forceinline__ void ev_weights(const EvictArgs& A, int64_t unit, int64_t rows, int64_t block) {
    float* dst = A.dst_weights + unit * A.dst_seq;
    const float* src = A.kept_weights + unit * A.most;
    const int64_t t0 = block * 2048, t1 = min(t0 + 2048, A.dst_seq);
    for (int64_t t = t0 + threadIdx.x; t < t1; t += 256) dst[t] = t < rows ? src[t] : 0.0f;
}

// blocks: the tiles of kept tokens of a head, then pieces of its weights
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_gather(EvictArgs A, uint8_t* dst, int64_t dst_seq_bytes, int64_t dst_head_bytes) {
    __shared__ int from[KV8_TILE];
    const int tile = blockIdx.x, h = blockIdx.y, seq = blockIdx.z;
    const int64_t unit = (int64_t)seq * A.nkv + h;
    const int64_t rows = A.rows[unit];
    if (tile >= A.gather_blocks) {  // (uniform)
        ev_weights(A, unit, rows, tile - A.gather_blocks);
        return;
    }
    if (tile == 0 && h == 0 && threadIdx.x == 0 && A.dst_lens) A.dst_lens[seq] = (int)rows;
    const int64_t t0 = (int64_t)tile * KV8_TILE;
    const int n = (int)min((int64_t)KV8_TILE, rows - t0);
    if (n <= 0) return;  // (uniform)
    const int* list = A.list + unit * A.list_stride + t0;
    if (A.in_place && list[n - 1] == t0 + n - 1) return;  // (uniform) the list ascends: nothing up to here moves
    if (threadIdx.x < n) from[threadIdx.x] = list[threadIdx.x];
    __syncthreads();
    ev_tile<HD>(dst + seq * dst_seq_bytes + h * dst_head_bytes + tile * aeth_kv8_tile_bytes(HD),
                A.cache + seq * A.seq_bytes + (int64_t)h * A.tiles * aeth_kv8_tile_bytes(HD), from, n);
}

// in place: the gathered tiles from the workspace
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_put_back(EvictArgs A, const uint8_t* stage, int64_t stage_seq_bytes, int64_t stage_head_bytes) {
    __shared__ int from[KV8_TILE];
    constexpr int64_t TB = aeth_kv8_tile_bytes(HD);
    const int tile = blockIdx.x, h = blockIdx.y, seq = blockIdx.z;
    const int64_t unit = (int64_t)seq * A.nkv + h, rows = A.rows[unit], t0 = (int64_t)tile * KV8_TILE;
    const int n = (int)min((int64_t)KV8_TILE, rows - t0);
    if (n <= 0) return;  // (uniform)
    const int* list = A.list + unit * A.list_stride + t0;
    if (list[n - 1] == t0 + n - 1) return;  // (uniform) as above
    const uint8_t* src = stage + seq * stage_seq_bytes + h * stage_head_bytes + tile * TB;
    uint8_t* dst = A.dst + seq * A.dst_seq_bytes + ((int64_t)h * A.dst_tiles + tile) * TB;
    if (n == KV8_TILE) {
        for (int64_t i = threadIdx.x; i < TB / 16; i += 256) ((uint4*)dst)[i] = ((const uint4*)src)[i];
        return;
    }
    if (threadIdx.x < n) from[threadIdx.x] = threadIdx.x;
    __syncthreads();
    ev_tile<HD>(dst, src, from, n);
}

// the workspace's parts, each 16-byte aligned: bytes from its start
struct EvictWs {
    int64_t list, weights, stage, end;
};
bool ev_ws(int64_t seqs, int64_t nkv, int64_t hd, int64_t most, bool in_place, EvictWs& W) {
    const int64_t units = seqs * nkv;  // below 2^32
    int64_t all, tiles;
    if (!aeth_mul_ok(units, most, &all) || !aeth_mul_ok(units * aeth_cdiv(most, KV8_TILE), aeth_kv8_tile_bytes((int)hd), &tiles) ||
        all > (int64_t)1 << 58 || tiles > (int64_t)1 << 60)
        return false;
    W.list = aeth_cdiv(4 * units, 16) * 16;
    W.weights = W.list + aeth_cdiv(4 * all, 16) * 16;
    W.stage = W.weights + aeth_cdiv(4 * all, 16) * 16;
    W.end = W.stage + (in_place ? tiles : 0);
    return true;
}

template <int HD>
int ev_launch(EvictArgs A, int64_t seqs, uint8_t* stage, hipStream_t s) {
    hipLaunchKernelGGL(k_kv8_select, dim3((unsigned)A.nkv, (unsigned)seqs), dim3(SEL), 0, s, A);
    AETH_LAUNCH_CHECK();
    const int64_t weight_blocks = A.dst_weights ? aeth_cdiv(A.dst_seq, 2048) : 0;
    const int64_t head = (int64_t)A.gather_blocks * aeth_kv8_tile_bytes(HD);
    const dim3 grid((unsigned)(A.gather_blocks + weight_blocks), (unsigned)A.nkv, (unsigned)seqs);
    if (stage) hipLaunchKernelGGL(k_kv8_gather<HD>, grid, dim3(256), 0, s, A, stage, head * A.nkv, head);
    else hipLaunchKernelGGL(k_kv8_gather<HD>, grid, dim3(256), 0, s, A, A.dst, A.dst_seq_bytes, A.dst_tiles * aeth_kv8_tile_bytes(HD));
    AETH_LAUNCH_CHECK();
    if (stage) {
        hipLaunchKernelGGL(k_kv8_put_back<HD>, dim3((unsigned)A.gather_blocks, (unsigned)A.nkv, (unsigned)seqs), dim3(256), 0, s, A, stage, head * A.nkv, head);
        AETH_LAUNCH_CHECK();
    }
    return AETH_OK;
}

bool apart(const void* a, int64_t na, const void* b, int64_t nb) {
    return (uintptr_t)a + (uint64_t)na <= (uintptr_t)b || (uintptr_t)b + (uint64_t)nb <= (uintptr_t)a;
}

int evict(const char* what, const void* cache, int64_t stride, const float* weights, const int* lens, int64_t seqs, int64_t nkv, int64_t hd,
          int64_t max_seq, int64_t max_len, int64_t keep, int64_t first, int64_t recent, void* dst, int64_t dst_stride, float* dst_weights,
          int64_t dst_seq, int* dst_lens, int* kept, void* ws, int64_t ws_bytes, hipStream_t s) {
    if (!cache || !weights || !dst || (((uintptr_t)cache | (uintptr_t)dst | (uintptr_t)ws) & 15) ||
        (((uintptr_t)weights | (uintptr_t)dst_weights | (uintptr_t)dst_lens | (uintptr_t)kept) & 3))
        return aeth_set_error(AETH_EINVAL, "%s: bad argument (slices and workspace 16-byte aligned, the rest 4-byte)", what);
    const int64_t bytes = aeth_kv8_layer_bytes(nkv, hd, max_seq), dst_bytes = aeth_kv8_layer_bytes(nkv, hd, dst_seq);
    if (bytes < 0 || dst_bytes < 0)
        return aeth_set_error(aeth_kv8_head_dim(hd) ? AETH_EINVAL : AETH_EUNSUPPORTED, "%s: bad shape (%lld heads of %lld, slices of %lld and %lld)", what,
                              (long long)nkv, (long long)hd, (long long)max_seq, (long long)dst_seq);
    if (max_len < 0 || max_len > max_seq || keep < 0 || first < 0 || recent < 0 || first > keep || recent > keep - first ||
        std::min(keep, max_len) > dst_seq)
        return aeth_set_error(AETH_EINVAL, "%s: %lld of %lld tokens kept (the first %lld and last %lld) in slices of %lld and %lld", what, (long long)keep,
                              (long long)max_len, (long long)first, (long long)recent, (long long)max_seq, (long long)dst_seq);
    int64_t all, dst_all, w_all, dw_all;
    if (seqs < 0 || seqs > 65535 || stride < 0 || dst_stride < 0 || ((stride | dst_stride) & 15) || (seqs > 1 && (stride < bytes || dst_stride < dst_bytes)) ||
        !aeth_mul_ok(seqs, std::max(stride, bytes), &all) || !aeth_mul_ok(seqs, std::max(dst_stride, dst_bytes), &dst_all) ||
        !aeth_mul_ok(seqs * nkv, max_seq, &w_all) || !aeth_mul_ok(seqs * nkv, dst_seq, &dw_all) || w_all > INT64_MAX / 4 || dw_all > INT64_MAX / 4)
        return aeth_set_error(AETH_EINVAL, "%s: %lld sequences %lld and %lld bytes apart", what, (long long)seqs, (long long)stride, (long long)dst_stride);
    const bool in_place = dst == cache;
    if (in_place ? dst_seq != max_seq || (seqs > 1 && dst_stride != stride) : !apart(cache, all, dst, dst_all))
        return aeth_set_error(AETH_EINVAL, "%s: the slices overlap, or are the same with another length or stride", what);
    if (dst_weights && (dst_weights == weights ? dst_seq != max_seq : !apart(weights, 4 * w_all, dst_weights, 4 * dw_all)))
        return aeth_set_error(AETH_EINVAL, "%s: the weights overlap, or are the same with another length", what);
    const int64_t most = std::min(keep, max_len);
    // workgroups of 256 threads within the grid's 2^32
    if (aeth_cdiv(most, KV8_TILE) + aeth_cdiv(dst_seq, 2048) > (int64_t)1 << 23)
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld tokens kept in one call", what, (long long)keep);
    EvictWs W;
    if (!ev_ws(seqs, nkv, hd, most, in_place, W)) return aeth_set_error(AETH_EINVAL, "%s: bad shape", what);
    if (seqs == 0) return AETH_OK;
    if (!ws || ws_bytes < W.end)
        return aeth_set_error(AETH_EINVAL, "%s: a workspace of %lld bytes (%lld given)", what, (long long)W.end, (long long)(ws ? ws_bytes : 0));
    EvictArgs A = {};
    A.cache = (const uint8_t*)cache;
    A.seq_bytes = stride;
    A.weights = weights;
    A.lens = lens;
    A.max_seq = max_seq;
    A.max_len = max_len;
    A.keep = keep;
    A.first = first;
    A.recent = recent;
    A.nkv = (int)nkv;
    A.tiles = (int)aeth_cdiv(max_seq, KV8_TILE);
    A.dst = (uint8_t*)dst;
    A.dst_seq_bytes = dst_stride;
    A.dst_seq = dst_seq;
    A.dst_tiles = (int)aeth_cdiv(dst_seq, KV8_TILE);
    A.dst_weights = dst_weights;
    A.dst_lens = dst_lens;
    A.rows = (int*)ws;
    A.list = kept ? kept : (int*)((char*)ws + W.list);
    A.list_stride = kept ? keep : most;
    A.kept_weights = (float*)((char*)ws + W.weights);
    A.most = most;
    A.gather_blocks = (int)std::max<int64_t>(1, aeth_cdiv(most, KV8_TILE));
    A.in_place = in_place;
    uint8_t* stage = in_place ? (uint8_t*)ws + W.stage : nullptr;
    if (hd == 64) return ev_launch<64>(A, seqs, stage, s);
    if (hd == 128) return ev_launch<128>(A, seqs, stage, s);
    return ev_launch<256>(A, seqs, stage, s);
}

}  // namespace

extern "C" AETH_API int64_t aeth_kv8_evict_ws_bytes(int64_t n_seqs, int64_t kv_heads, int64_t head_dim, int64_t max_len, int64_t keep, int in_place) {
    EvictWs W;
    if (n_seqs < 0 || n_seqs > 65535 || max_len < 0 || max_len > KV8_MAX_SEQ || keep < 0 || aeth_kv8_layer_bytes(kv_heads, head_dim, 1) < 0 ||
        !ev_ws(n_seqs, kv_heads, head_dim, std::min(keep, max_len), in_place != 0, W)) {
        aeth_set_error(AETH_EINVAL, "aeth_kv8_evict_ws_bytes: bad shape");
        return -1;
    }
    return W.end;
}

extern "C" AETH_API int aeth_kv8_evict(const void* d_layer, const float* d_weights, int64_t kv_heads, int64_t head_dim, int64_t max_seq, int64_t seq,
                                       int64_t keep, int64_t first, int64_t recent, void* d_dst, float* d_dst_weights, int64_t dst_seq,
                                       int32_t* d_kept, void* d_ws, int64_t ws_bytes, void* stream) {
    return evict("aeth_kv8_evict", d_layer, 0, d_weights, nullptr, 1, kv_heads, head_dim, max_seq, seq, keep, first, recent, d_dst, 0, d_dst_weights,
                 dst_seq, nullptr, d_kept, d_ws, ws_bytes, (hipStream_t)stream);
}

extern "C" AETH_API int aeth_kv8_evict_batch(const void* d_layers, int64_t layer_stride, const float* d_weights, const int32_t* d_lens, int64_t n_seqs,
                                             int64_t kv_heads, int64_t head_dim, int64_t max_seq, int64_t max_len, int64_t keep, int64_t first,
                                             int64_t recent, void* d_dst, int64_t dst_stride, float* d_dst_weights, int64_t dst_seq,
                                             int32_t* d_dst_lens, int32_t* d_kept, void* d_ws, int64_t ws_bytes, void* stream) {
    const char* what = "aeth_kv8_evict_batch";
    if (!d_lens || ((uintptr_t)d_lens & 3)) return aeth_set_error(AETH_EINVAL, "%s: bad argument (lengths)", what);
    return evict(what, d_layers, layer_stride, d_weights, d_lens, n_seqs, kv_heads, head_dim, max_seq, max_len, keep, first, recent, d_dst, dst_stride,
                 d_dst_weights, dst_seq, d_dst_lens, d_kept, d_ws, ws_bytes, (hipStream_t)stream);
}
