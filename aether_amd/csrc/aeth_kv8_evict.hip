// Eviction from the 8-bit cache (aeth_kv8.hpp) by the weight that each token has received.
//
// Of a head's len tokens `keep` stay: the first `first`, the last `recent`, and of the others the
// keep - first - recent of largest weight, the lower slot before the higher where weights are equal
// (NaN is below every number, -0 equals 0). They keep their order, their codes and their scales: a kept
// token stands for the same values as before. Three steps: the list of kept slots by head (k_kv8_select; k_kv8_count, k_kv8_number),
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

// sums of the values of a wave's lanes up to and with each
__device__ __forceinline__ uint32_t ev_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8: within rows of 16
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}

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
    int* rows;             // (the lengths may be overwritten before the last step)
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

// Weights as whole numbers in their order: NaN 1, -Inf 0x007FFFFF, +Inf 0xFF800000. What stays in any case has EV_STAYS, no slot 0,
// so that the kept ones are the `keep` largest.
constexpr uint32_t EV_STAYS = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t ev_key(float w) {
    const float y = w + 0.0f;  // -0 + 0 is 0
    const uint32_t f = __float_as_uint(y);
    return y != y ? 1u : f ^ ((uint32_t)((int)f >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint32_t ev_rank(uint64_t lanes) {  // of them those before this lane
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}

constexpr int SEL = 1024;             // threads of a selection
constexpr int NEAR = 32, FAR = 8;     // weights a thread holds: of a head in one workgroup, in many

struct EvictLds {
    __attribute__((aligned(16))) uint32_t hist[2048][4];  // a copy for every fourth lane: weights fill few bins, and lanes of one wait for each other
    uint32_t part[2][SEL / 64], sums[2][SEL / 64], found[3];
};

// f(0) .. f(J - 1) and on to a multiple of 4, four at a time (a jump over each of the others would fetch its code)
template <int PER, class F>
__device__ __forceinline__ void ev_each(int J, F&& f) {
#pragma unroll
    for (int g = 0; g < PER; g += 4) {
        if (g >= J) break;  // (uniform)
#pragma unroll
        for (int j = 0; j < 4; j++) f(g + j);
    }
}

// The weights of a piece of a head and their keys in a workgroup's registers: a wave has 64·J consecutive ones, lane l and register j
// 64·j + l of them, so that a rank among them is a count of bits.
template <int PER>
struct EvictHeld {
    float v[PER];
    uint32_t key[PER];
    int J, first;  // registers in use, the lane's slot in register 0
    __device__ __forceinline__ void load(const float* w, int base, int end) {  // slots from base on, below end
        J = (min(SEL * PER, end - base) + SEL - 1) / SEL;
        first = base + 64 * J * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + (threadIdx.x & 63);
        ev_each<PER>(J, [&](int j) { v[j] = w[(uint32_t)min(first + 64 * j, end - 1)]; });
    }
    __device__ __forceinline__ void keys(int lo, int hi, int end) {  // [lo, hi): the slots to choose from
        const int from = first - (threadIdx.x & 63), stop = min(end, from + 64 * J);
        ev_each<PER>(J, [&](int j) {
            key[j] = ev_key(v[j]);
            if (from + 64 * j < lo || from + 64 * j + 64 > min(hi, stop)) {  // (uniform)
                const int t = first + 64 * j;
                key[j] = t >= stop ? 0u : t < lo || t >= hi ? EV_STAYS : key[j];
            }
        });
    }
};

// What is known of the last key that stays: its first `done` bits, and how many to take of the keys that have them. `bits` more in the next pass; 0:
// keys above `last` stay, and `need` of those equal to it.
struct EvictState {
    uint32_t prefix, need, last;
    int done, bits;
};
__device__ __forceinline__ EvictState ev_start(int64_t keep) { return {0, (uint32_t)keep, 0, 0, 11}; }

__device__ __forceinline__ void ev_clear(EvictLds& L) {
    for (int i = threadIdx.x; i < 2048; i += SEL) *(uint4*)L.hist[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
}
// Counts keys that begin as is known by their next bits. (No slot's key counts too where a workgroup has all of a head: it is the lowest, and fewer
// stay than there are slots.)
template <int PER>
__device__ __forceinline__ void ev_count(const EvictState& S, const EvictHeld<PER>& H, EvictLds& L) {
    const int shift = 32 - S.done - S.bits;
    const uint32_t low = S.done > 0 ? S.prefix << S.bits : 0;
    uint32_t* mine = &L.hist[0][threadIdx.x & 3];
    ev_each<PER>(H.J, [&](int j) {
        const uint32_t bin = (H.key[j] >> shift) - low;
        if (bin < 1u << S.bits && (PER == NEAR || H.key[j] != 0)) atomicAdd(mine + 4 * bin, 1u);
    });
}
// the counts c1 of bin b + 1 and c0 of b = 2046 - 2·thread, of which one holds the need-th from the top: the pass done
__device__ __forceinline__ EvictState ev_find(EvictState S, uint32_t c1, uint32_t c0, EvictLds& L) {
    const int tid = threadIdx.x, wv = tid >> 6, b = 2046 - 2 * tid;
    const uint32_t x = ev_scan(c0 + c1);
    if ((tid & 63) == 63) L.part[0][wv] = x;
    __syncthreads();
    uint32_t above = x - c0 - c1;
#pragma unroll
    for (int i = 0; i < SEL / 64; i++) above += i < wv ? L.part[0][i] : 0;
    if (above < S.need && S.need <= above + c1) {
        L.found[0] = b + 1;
        L.found[1] = above;
        L.found[2] = c1;
    } else if (above + c1 < S.need && S.need <= above + c1 + c0) {
        L.found[0] = b;
        L.found[1] = above + c1;
        L.found[2] = c0;
    }
    __syncthreads();
    S.prefix = S.prefix << S.bits | L.found[0];
    S.need -= L.found[1];
    S.done += S.bits;
    S.last = S.prefix;
    S.bits = S.done == 22 ? 10 : S.done == 32 ? 0 : 11;
    if (L.found[2] == S.need) {  // (uniform) the whole bin; its lowest key is above 0: fewer stay than there are
        S.last = (S.prefix << (32 - S.done)) - 1;  // (done 32: a shift by 0)
        S.need = 0;
        S.bits = 0;
    }
    return S;
}

// Lists those of a piece that stay, behind `sures` above the last key and `equals` equal to it, and adds its own to them
template <int PER>
__device__ __forceinline__ void ev_number(const EvictState& S, const EvictHeld<PER>& H, EvictLds& L, int round, uint32_t& sures, uint32_t& equals, int* list,
                                          float* kw) {
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t ns = 0, ne = 0;  // (uniform) the wave's
    ev_each<PER>(H.J, [&](int j) {
        ns += (uint32_t)__popcll(__ballot(H.key[j] > S.last));
        ne += (uint32_t)__popcll(__ballot(H.key[j] == S.last));
    });
    if ((threadIdx.x & 63) == 0) {
        L.part[round][wv] = ns;
        L.sums[round][wv] = ne;
    }
    __syncthreads();  // (the other round's readers have passed the barrier before this one)
    uint32_t s0 = sures, e0 = equals;
#pragma unroll
    for (int i = 0; i < SEL / 64; i++) {
        const uint32_t a = L.part[round][i], b = L.sums[round][i];
        s0 += i < wv ? a : 0;
        e0 += i < wv ? b : 0;
        sures += a;
        equals += b;
    }
    ev_each<PER>(H.J, [&](int j) {
        const bool sure = H.key[j] > S.last, equal = H.key[j] == S.last;
        const uint64_t ms = __ballot(sure), me = __ballot(equal);
        const uint32_t e = e0 + ev_rank(me), at = s0 + ev_rank(ms) + min(e, S.need);
        if (sure || (equal && e < S.need)) {
            list[at] = H.first + 64 * j;
            kw[at] = H.v[j];
        }
        s0 += (uint32_t)__popcll(ms);
        e0 += (uint32_t)__popcll(me);
    });
}

// One workgroup a head of up to 32768 tokens. The last key that stays is found by up to three passes over the keys' bits (11, 11, 10) with
// counts in LDS (two, but for weights that are equal or nearly), the slots that stay numbered in a last one. What bounds it is instructions, on one
// CU a head: hence one word that says all of a token. 8 heads of 2500 tokens 7.0 µs, of 30000 19 (40 with weights read again in each pass
// and a scan over threads); 24 sequences' 4 heads of up to 4001 7.6.
__global__ void __launch_bounds__(SEL) k_kv8_select(EvictArgs A) {
    __shared__ EvictLds lds;
    const int seq = blockIdx.y, len = (int)ev_len(A, seq);
    const int64_t unit = (int64_t)seq * A.nkv + blockIdx.x;
    const float* w = A.weights + unit * A.max_seq;
    int* list = A.list + unit * A.list_stride;
    float* kw = A.kept_weights + unit * A.most;
    if (threadIdx.x == 0) A.rows[unit] = (int)min((int64_t)len, A.keep);
    if (len <= A.keep) {  // (uniform) all stay
        for (int t = threadIdx.x; t < len; t += SEL) {
            list[t] = t;
            kw[t] = w[t];
        }
        return;
    }
    if (A.keep == 0) return;  // (uniform)
    EvictHeld<NEAR> H;
    EvictState S = ev_start(A.keep);
    H.load(w, 0, len);
    ev_clear(lds);
    H.keys((int)A.first, len - (int)A.recent, len);
    while (S.bits > 0) {
        if (S.done > 0) ev_clear(lds);
        ev_count(S, H, lds);
        __syncthreads();
        const int b = 2046 - 2 * threadIdx.x;
        const uint4 h1 = *(const uint4*)lds.hist[b + 1], h0 = *(const uint4*)lds.hist[b];
        S = ev_find(S, h1.x + h1.y + h1.z + h1.w, h0.x + h0.y + h0.z + h0.w, lds);
    }
    uint32_t sures = 0, equals = 0;
    ev_number(S, H, lds, 0, sures, equals, list, kw);
}

// More tokens: many workgroups a head, a chunk of its slots each, and a launch for each pass. The workgroups of a pass leave their counts in memory,
// those of the next one add all of them up and go on from there, each for itself; the last launch knows from the counts how many stay before its chunk.
// 8 heads of 131000 tokens: 5 + 7 + 8 + 15 µs; one workgroup a head, which reads its weights again in each pass, 112.
struct EvictFar {
    uint32_t* hist;   // [3 passes][units][chunks][2048]
    uint32_t* state;  // [2][units][4]: behind the first pass, the second
    int64_t units;
    int chunk, chunks;  // slots of a chunk, a multiple of 8192; chunks of max_len slots
};
__device__ __forceinline__ const uint32_t* ev_counts(const EvictFar& F, int pass, int64_t unit, int c) {
    return F.hist + ((pass * F.units + unit) * F.chunks + c) * 2048;
}
__device__ __forceinline__ EvictState ev_resolve(const EvictState& S, const EvictFar& F, int pass, int64_t unit, int live, EvictLds& L) {
    uint32_t c1 = 0, c0 = 0;
#pragma unroll 4
    for (int c = 0; c < live; c++) {
        const uint2 n = *(const uint2*)(ev_counts(F, pass, unit, c) + 2046 - 2 * threadIdx.x);
        c0 += n.x;
        c1 += n.y;
    }
    return ev_find(S, c1, c0, L);
}
__device__ __forceinline__ void ev_keep_state(const EvictFar& F, int pass, int64_t unit, const EvictState& S) {
    if (blockIdx.x != 0 || threadIdx.x != 0) return;
    *(uint4*)(F.state + (pass * F.units + unit) * 4) = make_uint4(S.prefix, S.need, S.last, (uint32_t)(S.done << 8 | S.bits));
}
__device__ __forceinline__ EvictState ev_state(const EvictFar& F, int pass, int64_t unit) {
    const uint4 s = *(const uint4*)(F.state + (pass * F.units + unit) * 4);
    return {s.x, s.y, s.z, (int)(s.w >> 8), (int)(s.w & 255)};
}

template <int PASS>
__global__ void __launch_bounds__(SEL) k_kv8_count(EvictArgs A, EvictFar F) {
    __shared__ EvictLds lds;
    const int seq = blockIdx.z, len = (int)ev_len(A, seq), s0 = (int)blockIdx.x * F.chunk, s1 = min(s0 + F.chunk, len), live = (len + F.chunk - 1) / F.chunk;
    if (s0 >= len || len <= A.keep || A.keep == 0) return;  // (uniform)
    const int64_t unit = (int64_t)seq * A.nkv + blockIdx.y;
    EvictState S = ev_start(A.keep);
    if constexpr (PASS == 1) S = ev_resolve(S, F, 0, unit, live, lds);
    if constexpr (PASS == 2) {
        S = ev_state(F, 0, unit);
        if (S.bits > 0) S = ev_resolve(S, F, 1, unit, live, lds);  // (uniform)
    }
    if constexpr (PASS > 0) ev_keep_state(F, PASS - 1, unit, S);
    if (S.bits == 0) return;  // (uniform)
    EvictHeld<FAR> H;
    ev_clear(lds);
    for (int base = s0; base < s1; base += SEL * FAR) {
        H.load(A.weights + unit * A.max_seq, base, s1);
        H.keys((int)A.first, len - (int)A.recent, s1);
        ev_count(S, H, lds);
    }
    __syncthreads();
    uint32_t* out = F.hist + ((PASS * F.units + unit) * F.chunks + blockIdx.x) * 2048;
    for (int i = threadIdx.x; i < 2048; i += SEL) {
        const uint4 n = *(const uint4*)lds.hist[i];
        out[i] = n.x + n.y + n.z + n.w;
    }
}

__global__ void __launch_bounds__(SEL) k_kv8_number(EvictArgs A, EvictFar F) {
    __shared__ EvictLds lds;
    const int seq = blockIdx.z, len = (int)ev_len(A, seq), s0 = (int)blockIdx.x * F.chunk, s1 = min(s0 + F.chunk, len), live = (len + F.chunk - 1) / F.chunk;
    const int tid = threadIdx.x;
    const int64_t unit = (int64_t)seq * A.nkv + blockIdx.y;
    const float* w = A.weights + unit * A.max_seq;
    int* list = A.list + unit * A.list_stride;
    float* kw = A.kept_weights + unit * A.most;
    if (blockIdx.x == 0 && tid == 0) A.rows[unit] = (int)min((int64_t)len, A.keep);
    if (len <= A.keep) {  // (uniform) all stay
        for (int t = s0 + tid; t < s1; t += SEL) {
            list[t] = t;
            kw[t] = w[t];
        }
        return;
    }
    if (s0 >= len || A.keep == 0) return;  // (uniform)
    EvictState S = ev_state(F, 1, unit);
    if (S.bits > 0) S = ev_resolve(S, F, 2, unit, live, lds);  // (uniform)
    // before the chunk: keys of a higher bin in some pass, and of the last pass' own bin where all of it stays, or the equal ones
    uint32_t sures = 0, equals = 0;
    for (int pass = 0; pass < 3; pass++) {
        const int known = pass < 2 ? 11 * (pass + 1) : 32;
        if (known > S.done) break;  // (uniform)
        const uint32_t bin = S.prefix >> (S.done - known) & (pass < 2 ? 2047u : 1023u);
        const bool ends = known == S.done;
        for (int c = 0; c < (int)blockIdx.x; c++) {
            const uint2 n = *(const uint2*)(ev_counts(F, pass, unit, c) + 2 * tid);
            const uint32_t b = 2 * tid;
            sures += (b > bin || (ends && S.need == 0 && b == bin) ? n.x : 0) + (b + 1 > bin || (ends && S.need == 0 && b + 1 == bin) ? n.y : 0);
            if (ends && S.need > 0) equals += b == bin ? n.x : b + 1 == bin ? n.y : 0;
        }
    }
    sures = ev_scan(sures);
    equals = ev_scan(equals);
    __syncthreads();  // (ev_resolve's readers)
    if ((tid & 63) == 63) {
        lds.part[1][tid >> 6] = sures;
        lds.sums[1][tid >> 6] = equals;
    }
    __syncthreads();
    sures = equals = 0;
#pragma unroll
    for (int i = 0; i < SEL / 64; i++) {
        sures += lds.part[1][i];
        equals += lds.sums[1][i];
    }
    EvictHeld<FAR> H;
    int round = 0;  // (the first writes part[0])
    for (int base = s0; base < s1; base += SEL * FAR, round ^= 1) {
        H.load(w, base, s1);
        H.keys((int)A.first, len - (int)A.recent, s1);
        ev_number(S, H, lds, round, sures, equals, list, kw);
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

// blocks: the tiles of kept tokens of a head, then pieces of its weights. Memory bounds it where much is kept: half of 64 sequences' 4096 tokens
// of 8 heads of 128 155 µs, 4.5 TB/s of what it touches (all rows of V, kept rows of K, both written); 2048 of 2500 tokens 7.5, the way from the
// list to the bytes. A lane takes bytes of four tokens that are a word of the destination: neighbours mostly share a source line.
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_gather(EvictArgs A, uint8_t* dst, int64_t dst_seq_bytes, int64_t dst_head_bytes) {
    __shared__ int from[KV8_TILE];
    const int tile = blockIdx.x, h = blockIdx.y, seq = blockIdx.z;
    const int64_t unit = (int64_t)seq * A.nkv + h;
    const int64_t rows = A.lens ? A.rows[unit] : A.most;
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

// in place: the gathered tiles from the workspace (the 64 sequences' 96 µs: 5.8 TB/s)
template <int HD>
__global__ void __launch_bounds__(256) k_kv8_put_back(EvictArgs A, const uint8_t* stage, int64_t stage_seq_bytes, int64_t stage_head_bytes) {
    __shared__ int from[KV8_TILE];
    constexpr int64_t TB = aeth_kv8_tile_bytes(HD);
    const int tile = blockIdx.x, h = blockIdx.y, seq = blockIdx.z;
    const int64_t unit = (int64_t)seq * A.nkv + h, rows = A.lens ? A.rows[unit] : A.most, t0 = (int64_t)tile * KV8_TILE;
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

// A head of many tokens is counted in at most 64 chunks
constexpr int64_t FAR_CHUNK = SEL * FAR, FAR_CHUNKS = 64;
bool ev_far(int64_t max_len) { return max_len > SEL * NEAR; }

// the workspace's parts, each 16-byte aligned: bytes from its start
struct EvictWs {
    int64_t list, weights, state, hist, stage, end;
};
bool ev_ws(int64_t seqs, int64_t nkv, int64_t hd, int64_t max_len, int64_t keep, bool in_place, EvictWs& W) {
    const int64_t units = seqs * nkv, most = std::min(keep, max_len);  // units below 2^32
    const int64_t chunks = ev_far(max_len) ? std::min(FAR_CHUNKS, aeth_cdiv(max_len, FAR_CHUNK)) : 0;
    int64_t all, tiles;
    if (!aeth_mul_ok(units, most, &all) || !aeth_mul_ok(units * aeth_cdiv(most, KV8_TILE), aeth_kv8_tile_bytes((int)hd), &tiles) ||
        all > (int64_t)1 << 58 || tiles > (int64_t)1 << 60)
        return false;
    W.list = aeth_cdiv(4 * units, 16) * 16;
    W.weights = W.list + aeth_cdiv(4 * all, 16) * 16;
    W.state = W.weights + aeth_cdiv(4 * all, 16) * 16;
    W.hist = W.state + (chunks > 0 ? 32 * units : 0);
    W.stage = W.hist + 3 * units * chunks * 2048 * 4;
    W.end = W.stage + (in_place ? tiles : 0);
    return true;
}

template <int HD>
int ev_launch(EvictArgs A, EvictFar F, int64_t seqs, uint8_t* stage, hipStream_t s) {
    if (ev_far(A.max_len)) {
        const dim3 grid((unsigned)F.chunks, (unsigned)A.nkv, (unsigned)seqs), block(SEL);
        hipLaunchKernelGGL(k_kv8_count<0>, grid, block, 0, s, A, F);
        hipLaunchKernelGGL(k_kv8_count<1>, grid, block, 0, s, A, F);
        hipLaunchKernelGGL(k_kv8_count<2>, grid, block, 0, s, A, F);
        hipLaunchKernelGGL(k_kv8_number, grid, block, 0, s, A, F);
    } else {
        hipLaunchKernelGGL(k_kv8_select, dim3((unsigned)A.nkv, (unsigned)seqs), dim3(SEL), 0, s, A);
    }
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
    int64_t all, dst_all, w_all, dw_all, k_all = 0;
    if (seqs < 0 || seqs > 65535 || stride < 0 || dst_stride < 0 || ((stride | dst_stride) & 15) || (seqs > 1 && (stride < bytes || dst_stride < dst_bytes)) ||
        !aeth_mul_ok(seqs, std::max(stride, bytes), &all) || !aeth_mul_ok(seqs, std::max(dst_stride, dst_bytes), &dst_all) ||
        (kept && !aeth_mul_ok(seqs * nkv, keep, &k_all)) || !aeth_mul_ok(seqs * nkv, max_seq, &w_all) || !aeth_mul_ok(seqs * nkv, dst_seq, &dw_all) ||
        k_all > INT64_MAX / 4 || w_all > INT64_MAX / 4 || dw_all > INT64_MAX / 4)
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
    if (!ev_ws(seqs, nkv, hd, max_len, keep, in_place, W)) return aeth_set_error(AETH_EINVAL, "%s: bad shape", what);
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
    EvictFar F = {};
    F.hist = (uint32_t*)((char*)ws + W.hist);
    F.state = (uint32_t*)((char*)ws + W.state);
    F.units = seqs * nkv;
    F.chunk = (int)(aeth_cdiv(max_len, FAR_CHUNKS * FAR_CHUNK) * FAR_CHUNK);
    F.chunks = (int)(max_len > 0 ? aeth_cdiv(max_len, F.chunk) : 0);
    if (hd == 64) return ev_launch<64>(A, F, seqs, stage, s);
    if (hd == 128) return ev_launch<128>(A, F, seqs, stage, s);
    return ev_launch<256>(A, F, seqs, stage, s);
}

}  // namespace

extern "C" AETH_API int64_t aeth_kv8_evict_ws_bytes(int64_t n_seqs, int64_t kv_heads, int64_t head_dim, int64_t max_len, int64_t keep, int in_place) {
    EvictWs W;
    if (n_seqs < 0 || n_seqs > 65535 || max_len < 0 || max_len > KV8_MAX_SEQ || keep < 0 || aeth_kv8_layer_bytes(kv_heads, head_dim, 1) < 0 ||
        !ev_ws(n_seqs, kv_heads, head_dim, max_len, keep, in_place != 0, W)) {
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
