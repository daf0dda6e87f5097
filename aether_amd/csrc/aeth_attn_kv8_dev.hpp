// Attention over the 8-bit cache (aeth_kv8.hpp): its kernels and the choice of its form, for the calls of aeth_attn_kv8.hip
// (sequences, chunks, batches) and of aeth_attn_kv8_serve.hip (a shared prefix, the weights that tokens receive). GQA, causal, with a sliding window.
//
// Query i of n stands at position p = len - n + i of a sequence of len tokens and sees the keys
// max(0, p - window + 1) .. p. A column is one (query, head): column x = i·G + head of the G query
// heads that share a KV head; 16 columns fill the int8 matrix product
//   Sᵀ[64 tokens][16] = K[64][hd] · Qᵀ,   Oᵀ[hd][16] += Vᵀ[hd][64] · Pᵀ
// on v_mfma_i32_16x16x64_i8. The codes are one operand as they stand. q and the probabilities enter
// as integers of 24 bits, three balanced base-256 digits d2·65536 + d1·256 + d0 with d in [-128, 127]:
// three int8 products whose i32 sums are exact. So
//  * a score carries q rounded to 2^-23 of its row's largest component (|q·2^e| in [2^22, 2^23)), as
//    keys are held to 2^-8 of theirs, and nothing else but the f32 roundings of its final products. More
//    digits would cost a third more products; where a fourth of q is 30 times larger and of the keys
//    30 times smaller it costs four times f32's error (4.7e-6 of the result over 2049 tokens), else none;
//  * p·sv (the probability times the token's V scale) is rounded to 2^-23 of the largest of its column
//    in a tile of 64 tokens, whatever the running maximum: neither a flat row nor a tile far below
//    the maximum loses bits. Tiles are summed in f32.
// Running maximum and sum in f32, in log2 units; the partials are rescaled only when some column's
// maximum grows by more than 2^8 (the result does not depend on which maximum is used).
// A masked key's score, probability and V scale are replaced by selects, so infinities and NaN there
// reach nothing; a visible token whose scale is NaN makes the columns that see it NaN.
#pragma once
#include <math.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "aeth_common.hpp"
#include "aeth_internal.hpp"
#include "aeth_kv8.hpp"
#include "aeth_ops_internal.hpp"

typedef int a8_i4 __attribute__((ext_vector_type(4)));
typedef float a8_f4 __attribute__((ext_vector_type(4)));

namespace {

struct A8 {
    const float* q;         // [seqs][n] rows of q_stride floats
    int64_t q_stride;
    const uint8_t* cache;
    int64_t seq_bytes;
    const int* lens;        // [seqs]: len = lens[seq] + len_add, clamped to [0, max_len]; nullptr: max_len
    int len_add, max_len;
    int n, nq, nkv, G, cols;  // queries, query heads, KV heads, query heads a KV head, n·G
    int tiles;              // tiles a head's slice holds
    int window;             // 0: none
    int ncb, chunks, tpc;   // column blocks, chunks of tpc tiles
    float* out;             // [seqs][n][nq·hd]
    float* ws;              // partials when chunks > 1
    int qvec, ovec;         // q rows / out 16-byte aligned
    // a decode step (A8_STEP): q is q | k | v unrotated, lens the cache fill, len_add 1
    const int* pos;         // device position of the token
    const float *sin_t, *cos_t;
    int64_t max_seq;
    // a prefix that every row sees (A8_FLAT): the rows are sequences of own_lens tokens behind it, clamped to [0, own_max]
    const int* own_lens;
    int own_max;
    float* stat;            // A8_STAT: [seqs][nkv][cols] maximum and 1 / sum of each column
    float* scores;          // A8_SCORE: [seqs][nkv][cols][64·score_tiles], from key 0 on
    int score_tiles;
};

// What a kernel does beside or instead of its plain form
enum {
    A8_STEP = 1,   // a decode step's token with it
    A8_FLAT = 2,   // no order: every column sees the keys [0, max_len), those in the window of its sequence
    A8_PART = 4,   // partials also where there is one chunk
    A8_STAT = 8,   // columns' maxima and 1 / sums to A.stat (where chunks are joined, by the join)
    A8_SCORE = 16, // the scores, in log2 units, of the tiles that some column of the block sees, to A.scores
};

// f(0) .. f(N - 1), each with its number as a constant
template <int... I, class F>
__device__ __forceinline__ void a8_unroll_(std::integer_sequence<int, I...>, F&& f) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void a8_unroll(F&& f) {
    a8_unroll_(std::make_integer_sequence<int, N>{}, f);
}

// lane I of the lane's row of 16: an operand modifier of the instruction that uses it
template <int I>
__device__ __forceinline__ float a8_row(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x150 + I, 0xF, 0xF, true));  // row_newbcast
}

// 2^j of the largest j with |x|·2^j <= 0x7F7F00 for |x| <= mx (three balanced digits), as its exponent;
// 0 for mx = 0, infinite or NaN
__device__ __forceinline__ int a8_exponent(float mx) {
    if (!(mx > 0.0f && mx < INFINITY)) return 0;
    int e;
    (void)frexpf(mx, &e);
    int j = min(23 - e, 126);
    if (ldexpf(mx, j) > 8355584.0f) j--;
    return max(j, -126);
}
__device__ __forceinline__ float a8_pow2(int j) { return __int_as_float((127 + j) << 23); }

// Four words X + 0x8080 (24 bits and more) → the words of their digits: bytes 0 and 1 are digit + 128, byte 2 is the digit (of X >= 0)
__device__ __forceinline__ void a8_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t& d0, uint32_t& d1, uint32_t& d2) {
    const uint32_t p = __builtin_amdgcn_perm(b, a, 0x05010400u), q = __builtin_amdgcn_perm(d, c, 0x05010400u);
    const uint32_t s = __builtin_amdgcn_perm(b, a, 0x0C0C0602u), t = __builtin_amdgcn_perm(d, c, 0x0C0C0602u);
    d0 = __builtin_amdgcn_perm(q, p, 0x05040100u) ^ 0x80808080u;
    d1 = __builtin_amdgcn_perm(q, p, 0x07060302u) ^ 0x80808080u;
    d2 = __builtin_amdgcn_perm(t, s, 0x05040100u);
}
// ... of four integers, |X| <= 0x7F7F00
__device__ __forceinline__ void a8_digits(int a, int b, int c, int d, uint32_t& d0, uint32_t& d1, uint32_t& d2) {
    a8_bytes((uint32_t)a + 0x808080u, (uint32_t)b + 0x808080u, (uint32_t)c + 0x808080u, (uint32_t)d + 0x808080u, d0, d1, d2);
    d2 ^= 0x80808080u;
}

// Three digits' products, d2·65536 + d1·256 + d0, as f32: the low ones' sum starts from the bits of 1.5·2^23 and so is a
// float as it stands (|d0| <= 128·127·256 < 2^22), the middle ones' from -1.5·2^23 / 256, which the fused addition takes out exactly
#define A8_START0 (a8_i4){0x4B400000, 0x4B400000, 0x4B400000, 0x4B400000}
#define A8_START1 (a8_i4){-49152, -49152, -49152, -49152}
__device__ __forceinline__ float a8_join(int d0, int d1, int d2) { return fmaf((float)((d2 << 8) + d1), 256.0f, __int_as_float(d0)); }

// the first key that column's sequence sees of a prefix: its window ends behind its own tokens
__device__ __forceinline__ int a8_flat_lo(const A8& A, int qi) { return A.max_len + min(max(A.own_lens[qi], 0), A.own_max) - A.window; }

__device__ __forceinline__ int a8_len(const A8& A, int seq) {
    if (!A.lens) return A.max_len;
    const int64_t l = (int64_t)A.lens[seq] + A.len_add;
    return (int)min(max(l, (int64_t)0), (int64_t)A.max_len);
}

// The tiles some column of columns [c0, c0 + count) sees: [beg, end)
template <int MODE = 0>
__device__ __forceinline__ void a8_tiles(const A8& A, int len, int c0, int count, int& beg, int& end) {
    if constexpr ((MODE & A8_FLAT) != 0) {  // an own token more moves the window on
        beg = A.window > 0 ? max(0, A.max_len - A.window) >> 6 : 0;
        end = (A.max_len + 63) >> 6;
        return;
    }
    const int i0 = c0 / A.G, i1 = min(c0 + count, A.cols) - 1;
    const int hi = len - A.n + i1 / A.G + 1;                                      // keys < hi
    const int lo = A.window > 0 ? max(0, len - A.n + i0 + 1 - A.window) : 0;
    beg = lo >> 6;
    end = hi > 0 ? (hi + 63) >> 6 : 0;
    if (end < beg) end = beg;
}

// Workgroup (KV head, column block of 16, chunk, sequence): its four waves take the chunk's tiles round robin,
// each with its own running softmax, and merge through LDS. 32 / 8 heads of 128: a token over 2049 positions 6.7 µs (one tile a
// wave: its loads and the chain from them to the output, beside 2.3 of an empty launch), over 131000 48 (5.7 TB/s, memory),
// 48 tokens over up to 4096 46 (4.6 TB/s: uneven lengths); 512 queries 17.9 (three instructions to join a
// score's digits, four for an output's, five to make a probability's, and two rounds of workgroups that live for two tiles a wave).
// A token's scales belong to one register of every lane (lane group g holds tokens 16j + 4g + r in registers
// 4j + r): lane i of a row of 16 holds the one of register i's token, and the multiplication takes it from there.
// STEP (HD = 128, one column block): a decode step's token with it. Each workgroup rotates q; the wave that takes the token's
// tile also rotates k, quantises k and v, stores them and puts the codes into the fragments it loaded.
template <int HD, int MODE>
__device__ __forceinline__ void a8_few(const A8& A, const int bx, const int seq, const int chunk, float (&po)[4][16][HD + 4], float (&pm)[4][16],
                                       float (&pl)[4][16], uint32_t (&fresh)[2][HD / 4]) {
    constexpr bool STEP = (MODE & A8_STEP) != 0, FLAT = (MODE & A8_FLAT) != 0, PART = (MODE & A8_PART) != 0;
    static_assert(!STEP || HD == 128, "a lane holds both halves of a rotated pair");
    constexpr int KS = HD / 64, DT = HD / 16;
    constexpr float TH = 8.0f;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = bx % A.nkv, cb = A.ncb - 1 - bx / A.nkv;  // late queries, the longest rows, first
    const int len = a8_len(A, seq);
    int beg, end;
    a8_tiles<MODE>(A, len, cb * 16, 16, beg, end);
    const int t0 = beg + chunk * A.tpc, t1 = min(t0 + A.tpc, end);
    if (t0 >= t1 && chunk > 0) return;  // (uniform) the merge leaves it out
    const uint8_t* head = A.cache + seq * A.seq_bytes + (int64_t)h * A.tiles * aeth_kv8_tile_bytes(HD);

    a8_i4 kf[4][KS], vf[DT];
    float sk, sv;
    // codes that one workgroup alone reads go past the caches (131000 tokens: 47.6 µs against 51.4)
    const bool once = A.ncb == 1;
    auto load = [&](int t) {
        const uint8_t* p = head + (int64_t)t * aeth_kv8_tile_bytes(HD);
        const int st = 16 * ((lane >> 2) & 3) + 4 * g + (lane & 3);
        sk = *(const float*)(p + 2 * KV8_TILE * HD + 4 * st);
        sv = *(const float*)(p + 2 * KV8_TILE * HD + 4 * (KV8_TILE + st));
        auto codes = [&](auto ld) {
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int s = 0; s < KS; s++) kf[j][s] = ld((const a8_i4*)(p + (16 * j + c) * HD + 64 * s + 16 * g));
#pragma unroll
            for (int dt = 0; dt < DT; dt++) vf[dt] = ld((const a8_i4*)(p + KV8_TILE * HD + (16 * dt + c) * KV8_TILE + 16 * g));
        };
        if (once) codes([](const a8_i4* a) { return __builtin_nontemporal_load(a); });
        else codes([](const a8_i4* a) { return *a; });
    };

    // the column: q (its loads go out first), the keys [lo, hi) it sees
    const int x = cb * 16 + c, xc = min(x, A.cols - 1), qi = xc / A.G;
    float qv[KS][16];
    {
        const float* src = A.q + ((int64_t)seq * A.n + qi) * A.q_stride + (int64_t)(h * A.G + xc % A.G) * HD + 16 * g;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                float4 y;
                if (A.qvec) y = *(const float4*)(src + 64 * s + e);
                else y = make_float4(src[64 * s + e], src[64 * s + e + 1], src[64 * s + e + 2], src[64 * s + e + 3]);
                qv[s][e] = y.x;
                qv[s][e + 1] = y.y;
                qv[s][e + 2] = y.z;
                qv[s][e + 3] = y.w;
            }
    }
    // STEP: the table's row; k and v of the token, a row of 16 lanes each, if this wave takes their tile
    const int slot = STEP ? A.lens[0] : -1, fresh_t = slot >> 6;
    const bool mine = STEP && slot >= 0 && slot < len && fresh_t >= t0 && fresh_t < t1 && ((fresh_t - t0) & 3) == w;  // (uniform)
    float sn[STEP ? 16 : 1], cs[STEP ? 16 : 1];
    float4 xa, xb, xs, xc4;
    const float *sin_r = nullptr, *cos_r = nullptr;
    if constexpr (STEP) {
        const int64_t p = min(max((int64_t)A.pos[0], (int64_t)0), A.max_seq - 1);
        sin_r = A.sin_t + p * (HD / 2);
        cos_r = A.cos_t + p * (HD / 2);
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            *(float4*)&sn[e] = *(const float4*)(sin_r + 16 * g + e);
            *(float4*)&cs[e] = *(const float4*)(cos_r + 16 * g + e);
        }
        if (mine) {
            const float* src = A.q + (int64_t)(A.nq + (lane >> 4 & 1) * A.nkv + h) * HD + 4 * c;
            xa = *(const float4*)src;
            xb = *(const float4*)(src + HD / 2);
            xs = *(const float4*)(sin_r + 4 * c);
            xc4 = *(const float4*)(cos_r + 4 * c);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (t0 + w < t1) load(t0 + w);
    __builtin_amdgcn_sched_barrier(0);
    float fresh_s = 0.0f;  // the scale of K (lanes of rows 0 and 2) or V (1 and 3)
    if constexpr (STEP) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float a = qv[0][e], b = qv[KS - 1][e];
            qv[0][e] = kv8_rot0(a, b, sn[e], cs[e]);
            qv[KS - 1][e] = kv8_rot1(a, b, sn[e], cs[e]);
        }
        if (mine) {
            const int v = lane >> 4 & 1;
            float4 ra = xa, rb = xb;
            kv8_rotate(ra, rb, xs, xc4);
            if (v) ra = xa, rb = xb;
            const Kv8Row q = kv8_quantise<HD>(ra, rb);
            fresh_s = q.scale;
            if (lane < 32) {
                fresh[v][c] = q.a;
                fresh[v][c + 16] = q.b;
                kv8_put<HD>((uint8_t*)head, slot, v, 4 * c, q);
            }
        }
    }
    a8_i4 qd[3][KS];  // q's digits
    float qs;
    {
        uint32_t mb = 0;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 16; e++) mb = max(mb, __float_as_uint(qv[s][e]) & 0x7FFFFFFFu);
        // over the four lane groups, as integers: a NaN's bits are above an infinity's
        const auto a = __builtin_amdgcn_permlane16_swap(mb, mb, false, false);
        mb = max(a[0], a[1]);
        const auto b = __builtin_amdgcn_permlane32_swap(mb, mb, false, false);
        mb = max(b[0], b[1]);
        const int e2 = a8_exponent(__uint_as_float(mb));
        const float f = a8_pow2(e2);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t d0, d1, d2;
                a8_digits((int)rintf(qv[s][4 * e] * f), (int)rintf(qv[s][4 * e + 1] * f), (int)rintf(qv[s][4 * e + 2] * f),
                          (int)rintf(qv[s][4 * e + 3] * f), d0, d1, d2);
                qd[0][s][e] = (int)d0;
                qd[1][s][e] = (int)d1;
                qd[2][s][e] = (int)d2;
            }
        // an infinity or NaN in q: every score NaN
        qs = mb >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : a8_pow2(-e2) * (1.4426950408889634f / sqrtf((float)HD));
    }
    const int hi = FLAT ? A.max_len : len - A.n + qi + 1;
    const int lo = A.window > 0 ? (FLAT ? a8_flat_lo(A, qi) : hi - A.window) : 0;
    // every column of the block sees the keys [all_lo, all_hi)
    const int all_hi = FLAT ? A.max_len : len - A.n + (cb * 16) / A.G + 1;
    const int all_lo = A.window > 0 ? (FLAT ? 0x7FFFFFFF : len - A.n + (min(cb * 16 + 16, A.cols) - 1) / A.G + 1 - A.window) : 0;
    float m = -INFINITY, l = 0.0f;
    a8_f4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = (a8_f4){0.0f, 0.0f, 0.0f, 0.0f};

    const a8_i4 start[3] = {A8_START0, A8_START1, {0, 0, 0, 0}};
    for (int t = t0 + w; t < t1; t += 4) {
        if (STEP && mine && t == fresh_t) {  // (uniform) the token's codes and scales in place of what was loaded from its slot
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's stores of them
            const int j = slot >> 4 & 3, r8 = 8 * (slot & 3);
            a8_i4 row[KS];
#pragma unroll
            for (int s = 0; s < KS; s++) row[s] = *(const a8_i4*)&fresh[0][16 * s + 4 * g];
            uint32_t byte[DT];
#pragma unroll
            for (int dt = 0; dt < DT; dt++) byte[dt] = fresh[1][4 * dt + (c >> 2)] >> (8 * (c & 3)) & 0xFFu;
            const bool k_here = c == (slot & 15), v_here = g == (slot >> 2 & 3);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (i != j) continue;  // (uniform)
#pragma unroll
                for (int s = 0; s < KS; s++) kf[i][s] = k_here ? row[s] : kf[i][s];
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const uint32_t x = ((uint32_t)vf[dt][i] & ~(0xFFu << r8)) | byte[dt] << r8;
                    vf[dt][i] = v_here ? (int)x : vf[dt][i];
                }
            }
            const float fk = __shfl(fresh_s, 0, 64), fv = __shfl(fresh_s, 16, 64);
            if ((slot & 63) == 16 * ((lane >> 2) & 3) + 4 * g + (lane & 3)) {
                sk = fk;
                sv = fv;
            }
        }
        {   // a V scale that is no number goes to the token's K scale: its scores are NaN where it is seen
            const bool fine = fabsf(sv) < INFINITY;
            sk = fine ? sk : __uint_as_float(0x7FC00000u);
            sv = fine ? sv : 0.0f;
        }
        float s[16];
        a8_unroll<4>([&](auto jj) {
            constexpr int j = jj;
            a8_i4 d[3];
#pragma unroll
            for (int p = 0; p < 3; p++) {
                d[p] = start[p];
#pragma unroll
                for (int ks = 0; ks < KS; ks++) d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[j][ks], qd[p][ks], d[p], 0, 0, 0);
            }
            a8_unroll<4>([&](auto rr) {
                constexpr int r = rr, i = 4 * j + r;
                s[i] = a8_join(d[0][r], d[1][r], d[2][r]) * a8_row<i>(sk);
            });
        });
        if (64 * t < all_lo || 64 * t + 64 > all_hi) {  // (uniform) some key is masked
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int key = 64 * t + 16 * (i >> 2) + 4 * g + (i & 3);
                s[i] = key >= lo && key < hi ? s[i] : -INFINITY;
            }
        }
        if constexpr ((MODE & A8_SCORE) != 0) {
            if (x < A.cols) {
                float* dst = A.scores + ((int64_t)(seq * A.nkv + h) * A.cols + x) * (64 * (int64_t)A.score_tiles) + 64 * (int64_t)t + 4 * g;
#pragma unroll
                for (int j = 0; j < 4; j++) *(a8_f4*)(dst + 16 * j) = (a8_f4){s[4 * j], s[4 * j + 1], s[4 * j + 2], s[4 * j + 3]} * qs;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
        mx = aeth_max_rows(mx) * qs;
        if (__any(mx > m + TH)) {  // (uniform)
            const float mn = fmaxf(m, mx), al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[dt] *= al;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.0f : m;  // every key masked so far: s is -Inf
        float wm = 0.0f, ps = 0.0f;
        a8_unroll<16>([&](auto at) {
            constexpr int i = at;
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i], qs, -ref));
            ps += p;
            s[i] = p * a8_row<i>(sv);
            wm = fmaxf(wm, s[i]);
        });
        l += ps;
        wm = aeth_max_rows(wm);
        if (!(wm < INFINITY)) l = __uint_as_float(0x7FC00000u);  // p (below 2^9) times V past f32: no number rather than a wrong one
        const int j2 = a8_exponent(wm);
        const float f = a8_pow2(j2), fi = a8_pow2(-j2);
        a8_i4 pd[3];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t y[4], d0, d1, d2;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = __float_as_uint(fmaf(s[4 * j + r], f, 8388608.0f + 0x8080));  // below 2^24: rounded to whole
            a8_bytes(y[0], y[1], y[2], y[3], d0, d1, d2);
            pd[0][j] = (int)d0;
            pd[1][j] = (int)d1;
            pd[2][j] = (int)d2;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            a8_i4 d[3];
#pragma unroll
            for (int p = 0; p < 3; p++) d[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[dt], pd[p], start[p], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) o[dt][r] = fmaf(a8_join(d[0][r], d[1][r], d[2][r]), fi, o[dt][r]);
        }
        if (t + 4 < t1) load(t + 4);
    }
    l = aeth_sum_rows(l);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) *(a8_f4*)&po[w][c][16 * dt + 4 * g] = o[dt];
    if (g == 0) {
        pm[w][c] = m;
        pl[w][c] = l;
    }
    __syncthreads();
    float* part = A.ws + ((int64_t)((seq * A.nkv + h) * A.ncb + cb) * A.chunks + chunk) * 16 * (HD + 2);
    for (int at = tid; at < 16 * HD / 4; at += 256) {
        const int cc = at / (HD / 4), d = 4 * (at % (HD / 4)), x = cb * 16 + cc;
        if (x >= A.cols) continue;
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < 4; v++) M = fmaxf(M, pm[v][cc]);
        float L = 0.0f;
        a8_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < 4; v++) {
            const float wt = pm[v][cc] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(pm[v][cc] - M);
            L += wt * pl[v][cc];
            acc += *(const a8_f4*)&po[v][cc][d] * wt;
        }
        if (PART || A.chunks > 1) {
            *(a8_f4*)(part + cc * HD + d) = acc;
            if (d == 0) {
                part[16 * HD + 2 * cc] = M;
                part[16 * HD + 2 * cc + 1] = L;
            }
            continue;
        }
        if constexpr ((MODE & A8_STAT) != 0)
            if (d == 0) *(float2*)(A.stat + 2 * ((int64_t)(seq * A.nkv + h) * A.cols + x)) = make_float2(M, 1.0f / L);
        acc = L == 0.0f ? (a8_f4){0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / L);  // a row that sees nothing: 0
        float* dst = A.out + ((int64_t)seq * A.n + x / A.G) * ((int64_t)A.nq * HD) + (int64_t)(h * A.G + x % A.G) * HD + d;
        if (A.ovec) *(a8_f4*)dst = acc;
        else dst[0] = acc[0], dst[1] = acc[1], dst[2] = acc[2], dst[3] = acc[3];
    }
}

// (a grid's first chunks, which every sequence has, first)
template <int HD, int MODE>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_attn8(A8 A) {
    __shared__ __attribute__((aligned(16))) float po[4][16][HD + 4];
    __shared__ float pm[4][16], pl[4][16];
    __shared__ __attribute__((aligned(16))) uint32_t fresh[2][HD / 4];  // A8_STEP: the token's codes of K and V
    a8_few<HD, MODE>(A, blockIdx.x, blockIdx.y, blockIdx.z, po, pm, pl, fresh);
}

// ── many columns: a prompt, or a chunk of one ─────────────────────────────
// The int8 form above spends more on joining digits than on the softmax itself: three instructions a score,
// four an output and tile of 64 tokens, five a probability. Here the codes become fp16 (exactly), once for a workgroup's
// 32·NW columns, on their way to LDS, and q and the probabilities are each two fp16 parts, x = hi + lo
// (22 significant bits), so that both products run on v_mfma_f32_32x32x16_f16 in two passes that share
// their f32 accumulators: nothing is left to join.
//  * q: x·2^-e below 2^15, lo's last place 2^-24: to 2^-23 of each component (the small ones to 2^-40 of the row's
//    largest).
//  * p·sv enters times a power of two of its column, which follows the largest such product the column has seen
//    (in [2^9, 2^15)): to 2^-23 of itself, or 2^-34 of that largest one where it is far smaller.
// Wave = 32 columns; Sᵀ = K·Qᵀ leaves a lane (column l%32, half h = l/32) the keys 8a + 4h + r of 32, which is
// the order in which V's operand takes its tokens (j = 2T + u, g = 2a + h of aeth_kv8.hpp), so the
// probabilities stay in their lanes. The next tile's codes are loaded a tile ahead, converted and stored in
// the other LDS buffer before this tile's products: one barrier a tile.
// 32 / 8 heads of 128: 4000 tokens 253 µs (0.52 PFLOP/s of the formula, 1.04 of the matrix units'), 250 over 20000 159 with its
// join. The matrix units are busy 49 % of the cycles, at 2.0 GHz, the vector units (their issue of matrix instructions with it)
// 46 %: of two waves a SIMD one is often waiting for the other's instruction to leave the issue port (35 % of the waves' time) or
// for LDS and the barrier (32 %). The two
// phases of two waves kept apart by barriers, another priority for one of them, K a step ahead and reads from LDS further
// ahead took as long or longer.
typedef _Float16 a8_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 a8_h4 __attribute__((ext_vector_type(4)));
typedef _Float16 a8_h2 __attribute__((ext_vector_type(2)));
typedef float a8_f2 __attribute__((ext_vector_type(2)));
typedef float a8_f16 __attribute__((ext_vector_type(16)));

// the larger of a column's two lanes
__device__ __forceinline__ float a8_max_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

// four signed bytes as fp16
__device__ __forceinline__ a8_h4 a8_half4(uint32_t w) {
    w ^= 0x80808080u;
    const a8_h2 k = {(_Float16)-1152.0f, (_Float16)-1152.0f};  // (0x64 | b) is 1024 + b
    const a8_h2 a = __builtin_bit_cast(a8_h2, __builtin_amdgcn_perm(0x64646464u, w, 0x07010700u)) + k;
    const a8_h2 b = __builtin_bit_cast(a8_h2, __builtin_amdgcn_perm(0x64646464u, w, 0x07030702u)) + k;
    return (a8_h4){a[0], a[1], b[0], b[1]};
}

// V's buffers: three spare a barrier a tile; two let two workgroups of four waves share a CU's LDS
constexpr int a8_vbufs(int nw) { return nw == 8 ? 3 : 2; }
constexpr int A8_KF = 1040;  // bytes from one K fragment to the next: eight threads of a row store to eight bank groups

template <int HD, int NW, int MODE>
__device__ __forceinline__ void a8_many(const A8& A, const int bx, const int seq, const int chunk, char (&kb)[2][HD / 8 * A8_KF],
                                        char (&vb)[a8_vbufs(NW)][HD * 128], float (&sc)[a8_vbufs(NW)][2 * KV8_TILE]) {
    constexpr bool FLAT = (MODE & A8_FLAT) != 0, PART = (MODE & A8_PART) != 0;
    constexpr int KS = HD / 16, DT = HD / 32, NT = 64 * NW, CH = 4 * HD / NT;
    static_assert(CH >= 1 && CH * NT == 4 * HD, "16-byte pieces of a plane a thread");
    constexpr int KF = A8_KF;
    constexpr float TH = 8.0f;
    constexpr int NB = a8_vbufs(NW);
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = bx % A.nkv, cb = A.ncb - 1 - bx / A.nkv;
    const int len = a8_len(A, seq);
    int beg, end;
    a8_tiles<MODE>(A, len, cb * 32 * NW, 32 * NW, beg, end);
    const int t0 = beg + chunk * A.tpc, t1 = min(t0 + A.tpc, end);
    if (t0 >= t1 && chunk > 0) return;  // (uniform) the merge leaves it out
    const uint8_t* head = A.cache + seq * A.seq_bytes + (int64_t)h * A.tiles * aeth_kv8_tile_bytes(HD);

    uint4 rk[CH], rv[CH];
    float rsk = 0.0f, rsv = 0.0f;
    auto fetch_k = [&](int t) {
        const uint8_t* p = head + (int64_t)t * aeth_kv8_tile_bytes(HD);
#pragma unroll
        for (int u = 0; u < CH; u++) rk[u] = *(const uint4*)(p + 16 * (tid + NT * u));
        if (tid < KV8_TILE) {
            rsk = *(const float*)(p + 2 * KV8_TILE * HD + 4 * tid);
            rsv = *(const float*)(p + 2 * KV8_TILE * HD + 4 * (KV8_TILE + tid));
        }
    };
    auto fetch_v = [&](int t) {
        const uint8_t* p = head + (int64_t)t * aeth_kv8_tile_bytes(HD) + KV8_TILE * HD;
#pragma unroll
        for (int u = 0; u < CH; u++) rv[u] = *(const uint4*)(p + 16 * (tid + NT * u));
    };
    auto stage_k = [&](int b, int b3) {  // token t, dimensions 16·ks .. + 15 → lanes t%32 and 32 + t%32 of fragment (t/32, ks)
#pragma unroll
        for (int u = 0; u < CH; u++) {
            const int at = tid + NT * u, t = at / KS, ks = at % KS;
            char* dst = kb[b] + ((t >> 5) * KS + ks) * KF + (t & 31) * 16;
            const a8_h4 x = a8_half4(rk[u].x), y = a8_half4(rk[u].y), z = a8_half4(rk[u].z), q = a8_half4(rk[u].w);
            *(a8_h8*)dst = (a8_h8){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
            *(a8_h8*)(dst + 512) = (a8_h8){z[0], z[1], z[2], z[3], q[0], q[1], q[2], q[3]};
        }
        // a V scale that is no number goes to the token's K scale: its scores are NaN where it is seen
        if (tid < KV8_TILE) {
            const bool fine = fabsf(rsv) < INFINITY;
            sc[b3][tid] = fine ? rsk : __uint_as_float(0x7FC00000u);
            sc[b3][KV8_TILE + tid] = fine ? rsv : 0.0f;
        }
    };
    auto stage_v = [&](int b) {  // dimension d, token group g = 2a + half → half of a lane's eight tokens of fragments (d/32, j)
#pragma unroll
        for (int u = 0; u < CH; u++) {
            const int at = tid + NT * u, d = at >> 2, g = at & 3;
            char* dst = vb[b] + (d >> 5) * 4096 + ((d & 31) + 32 * (g & 1)) * 16 + 8 * (g >> 1);
            *(a8_h4*)dst = a8_half4(rv[u].x);
            *(a8_h4*)(dst + 1024) = a8_half4(rv[u].y);
            *(a8_h4*)(dst + 2048) = a8_half4(rv[u].z);
            *(a8_h4*)(dst + 3 * 1024) = a8_half4(rv[u].w);
        }
    };
    if (t0 < t1) {
        fetch_k(t0);
        fetch_v(t0);
    }

    const int x0 = cb * 32 * NW + 32 * w, x = x0 + c, xc = min(x, A.cols - 1), qi = xc / A.G;
    const int hi = FLAT ? A.max_len : len - A.n + qi + 1;
    const int lo = A.window > 0 ? (FLAT ? a8_flat_lo(A, qi) : hi - A.window) : 0;
    // every column of the wave sees the keys [all_lo, all_hi)
    const int i0 = min(x0, A.cols - 1) / A.G, i1 = min(x0 + 31, A.cols - 1) / A.G;
    const int all_hi = FLAT ? A.max_len : len - A.n + i0 + 1;
    const int all_lo = A.window > 0 ? (FLAT ? 0x7FFFFFFF : len - A.n + i1 + 1 - A.window) : 0;
    a8_h8 qh[KS], ql[KS];
    float qs;
    {
        const float* src = A.q + ((int64_t)seq * A.n + qi) * A.q_stride + (int64_t)(h * A.G + xc % A.G) * HD + 8 * hf;
        float y[KS][8];
        uint32_t mb = 0;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            if (A.qvec) {
                const float4 a = *(const float4*)(src + 16 * ks), b = *(const float4*)(src + 16 * ks + 4);
                y[ks][0] = a.x; y[ks][1] = a.y; y[ks][2] = a.z; y[ks][3] = a.w;
                y[ks][4] = b.x; y[ks][5] = b.y; y[ks][6] = b.z; y[ks][7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) y[ks][e] = src[16 * ks + e];
            }
#pragma unroll
            for (int e = 0; e < 8; e++) mb = max(mb, __float_as_uint(y[ks][e]) & 0x7FFFFFFFu);
        }
        const auto a = __builtin_amdgcn_permlane32_swap(mb, mb, false, false);
        mb = max(a[0], a[1]);
        const int e2 = a8_exponent(__uint_as_float(mb)) - 8;  // the largest below 2^15
        const float f = a8_pow2(e2);
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = y[ks][e] * f;
                qh[ks][e] = (_Float16)v;
                ql[ks][e] = (_Float16)(v - (float)qh[ks][e]);
            }
        // an infinity or NaN in q: every score NaN
        qs = mb >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : a8_pow2(-e2) * (1.4426950408889634f / sqrtf((float)HD));
    }
    // m: the largest score so far, up to 2^TH stale. The step's probabilities are formed times 2^lf, as 2^(score - ref) with
    // ref = m - lf; lf keeps the largest p·sv so far (top, and o, times 2^lf) in [2^9, 2^15). l is of the p themselves.
    // A column's two lanes follow their own halves of the keys; where one of them finds its bound passed, both agree anew.
    float m = -INFINITY, limit = -INFINITY, l = 0.0f, top = 0.0f, ref = 0.0f;  // limit: the product that is a score of m + TH
    int lf = 0;
    a8_f16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = (a8_f16){};
    a8_f16 s = (a8_f16){}, sn = (a8_f16){};  // this step's scores, the next one's products as they form
    constexpr int EK = 16 / KS, EV = 8 / DT;  // scores beside a k-step's products, beside a value fragment's

    // A token's scale belongs to a register of every lane: lane i of a row of 16 holds the one of register i's token, and
    // the multiplication takes it from there (one LDS word a lane and step in place of sixteen)
    const int st = 8 * ((lane >> 2) & 3) + 4 * hf + (lane & 3);
    auto scales = [&](int b3, int T, int part) { return sc[b3][KV8_TILE * part + 32 * T + st]; };
    auto rescale = [&](float al) {
        l *= al;
        top *= al;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] *= al;
    };
    auto shift = [&](int d) {  // lf becomes lf + d
        const float al = a8_pow2(d);
        top *= al;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] *= al;
        lf += d;
        ref = (m == -INFINITY ? 0.0f : m) - (float)lf;
    };
    // s, times its K scales, is a step's scores: masks them and follows their maximum
    auto bound_scores = [&](int k0) {
        if (k0 < all_lo || k0 + 32 > all_hi) {  // (uniform) some key is masked
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int key = k0 + 8 * (i >> 2) + 4 * hf + (i & 3);
                s[i] = key >= lo && key < hi ? s[i] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
        if (__any(mx > limit)) {  // (uniform)
            const float mn = fmaxf(m, a8_max_halves(mx) * qs);
            rescale(mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn));
            m = mn;
            limit = (m + TH) / qs;
            ref = (m == -INFINITY ? 0.0f : m) - (float)lf;
        }
    };
    // One step of 32 keys whose scores stand in s: its probabilities beside the products of the next step's scores,
    // its values' products beside what turns those into scores. The two run on different units, and the SIMD's
    // other wave fills what one leaves.
    auto step = [&](int b3, int T, const char* kp, int nb3, int nT, auto between) {
        const float sv = scales(b3, T, 1);
        a8_h8 kf[2] = {*(const a8_h8*)kp, *(const a8_h8*)(kp + KF)};
        // p is below 2^(lf + TH + 1), lf at most 100: p·sv below 2^127 up to these V scales, and for any with lf at -10, from where
        // it goes up again as the products are seen (1 % of the time, whether it is ever so or not)
        if (__any(sv > 0x1p18f)) shift(min(0, -10 - lf));  // (uniform)
        sn = (a8_f16){};
        float wm = 0.0f, ps = 0.0f;
        auto add = [&](auto at) {
            constexpr int i = at;
            ps += s[i];
            s[i] *= a8_row<i>(sv);
            wm = fmaxf(wm, s[i]);
        };
        a8_unroll<KS>([&](auto ks) {
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks & 1], ql[ks], sn, 0, 0, 0);
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks & 1], qh[ks], sn, 0, 0, 0);
            if (ks + 2 < KS) kf[ks & 1] = *(const a8_h8*)(kp + (ks + 2) * KF);
            a8_unroll<EK>([&](auto e) {
                constexpr int i = EK * ks + e;
                s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], qs, -ref));
                if constexpr (ks > 0) add(std::integral_constant<int, i - EK>{});
            });
        });
        a8_unroll<EK>([&](auto e) { add(std::integral_constant<int, 16 - EK + e>{}); });
        l = fmaf(ps, a8_pow2(-lf), l);
        top = fmaxf(top, wm);
        if (__any(__float_as_uint(top) - 0x44000000u >= 0x03000000u)) {  // (uniform) not in [2^9, 2^15)
            top = a8_max_halves(top);
            // top·2^d in [2^10, 2^11), as far as p·2^lf keeps clear of overflow (p·sv above 2^-90)
            const int d = top > 0.0f ? min(max(min(max(a8_exponent(top) - 12 + lf, -120), 100) - lf, -126), 126) : 0;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] *= a8_pow2(d);
            shift(d);
        }
        between();
        const char* vp = vb[b3] + 2 * T * 1024 + lane * 16;
        a8_h8 vf[2] = {*(const a8_h8*)vp, *(const a8_h8*)(vp + 4096)}, ph[2], pl[2];
        const float sk = scales(nb3, nT, 0);
        auto part = [&](int i) {  // hi and lo of s[i] and s[i + 1]: one packed conversion, two mixed-precision subtractions
            const a8_h2 y = __builtin_convertvector((a8_f2){s[i], s[i + 1]}, a8_h2);
            ph[i >> 3][i & 7] = y[0];
            ph[i >> 3][(i & 7) + 1] = y[1];
            a8_h2 z;
            asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(z) : "v"(s[i]), "v"(y));
            asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(z) : "v"(s[i + 1]), "v"(y));
            pl[i >> 3][i & 7] = z[0];
            pl[i >> 3][(i & 7) + 1] = z[1];
        };
#pragma unroll
        for (int i = 0; i < 8; i += 2) part(i);
        a8_unroll<2 * DT>([&](auto f) {  // (token half u, dimensions dt)
            constexpr int u = f / DT, dt = f % DT, n = f + 2;
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[f & 1], pl[u], o[dt], 0, 0, 0);
            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[f & 1], ph[u], o[dt], 0, 0, 0);
            if (n < 2 * DT) vf[f & 1] = *(const a8_h8*)(vp + (n % DT) * 4096 + n / DT * 1024);
            a8_unroll<EV>([&](auto e) {
                constexpr int i = EV * f + e;
                if (f < DT && i % 2 == 0) part(i + 8);
                s[i] = sn[i] * a8_row<i>(sk);
            });
        });
    };
    if (t0 < t1) {
        stage_k(0, 0);
        stage_v(0);
        if (t0 + 1 < t1) {
            fetch_k(t0 + 1);
            fetch_v(t0 + 1);
        }
    }
    __syncthreads();
    if (t0 < t1) {  // the first step's scores
        const char* kp = kb[0] + lane * 16;
        const float sk = scales(0, 0, 0);
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const a8_h8 kf = *(const a8_h8*)(kp + ks * KF);
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[ks], sn, 0, 0, 0);
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[ks], sn, 0, 0, 0);
        }
        a8_unroll<16>([&](auto at) {
            constexpr int i = at;
            s[i] = sn[i] * a8_row<i>(sk);
        });
        bound_scores(64 * t0);
    }
    // One barrier a tile, between its two steps: the codes of the next tile are stored before it, to K's other buffer,
    // whose last readers were two steps back, and V's third, whose readers were three (of two: one, behind a second
    // barrier). Behind the chunk's last tile a step's "next" products are of what the other buffer holds, and are dropped.
    int b3 = 0;
    for (int t = t0; t < t1; t++) {
        const int b = (t - t0) & 1, n3 = b3 == NB - 1 ? 0 : b3 + 1;
        step(b3, 0, kb[b] + KS * KF + lane * 16, b3, 1, [&] {
            if (t + 1 < t1) {
                stage_k(b ^ 1, n3);
                stage_v(n3);
                if (t + 2 < t1) {
                    fetch_k(t + 2);
                    fetch_v(t + 2);
                }
            }
        });
        bound_scores(64 * t + 32);
        __syncthreads();
        step(b3, 1, kb[b ^ 1] + lane * 16, n3, 0, [] {});
        if (t + 1 < t1) bound_scores(64 * t + 64);
        if (NB == 2) __syncthreads();
        b3 = n3;
    }
    {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if (x >= A.cols) return;
    const float un = a8_pow2(-lf);
    if (PART || A.chunks > 1) {
        const int cc = 32 * w + c;
        float* part = A.ws + ((int64_t)((seq * A.nkv + h) * A.ncb + cb) * A.chunks + chunk) * (32 * NW) * (HD + 2);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int a = 0; a < 4; a++)
                *(a8_f4*)(part + cc * HD + 32 * dt + 8 * a + 4 * hf) =
                    (a8_f4){o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]} * un;
        if (hf == 0) {
            part[32 * NW * HD + 2 * cc] = m;
            part[32 * NW * HD + 2 * cc + 1] = l;
        }
        return;
    }
    if constexpr ((MODE & A8_STAT) != 0)
        if (hf == 0) *(float2*)(A.stat + 2 * ((int64_t)(seq * A.nkv + h) * A.cols + x)) = make_float2(m, 1.0f / l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    float* dst = A.out + ((int64_t)seq * A.n + x / A.G) * ((int64_t)A.nq * HD) + (int64_t)(h * A.G + x % A.G) * HD + 4 * hf;
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
            const a8_f4 y = (a8_f4){o[dt][4 * a], o[dt][4 * a + 1], o[dt][4 * a + 2], o[dt][4 * a + 3]} * inv * un;
            float* d = dst + 32 * dt + 8 * a;
            if (A.ovec) *(a8_f4*)d = y;
            else d[0] = y[0], d[1] = y[1], d[2] = y[2], d[3] = y[3];
        }
}

template <int HD, int NW, int MODE>
__global__ void __launch_bounds__(64 * NW, 2) k_attn8p(A8 A) {
    constexpr int NB = a8_vbufs(NW);
    __shared__ __attribute__((aligned(16))) char kb[2][HD / 8 * A8_KF];
    __shared__ __attribute__((aligned(16))) char vb[NB][HD * 128];
    __shared__ __attribute__((aligned(16))) float sc[NB][2 * KV8_TILE];
    a8_many<HD, NW, MODE>(A, blockIdx.x, blockIdx.y, blockIdx.z, kb, vb, sc);
}

// Joins the chunks of one column (of blocks of cw): 256 threads, four dimensions each of every 1024/hd-th chunk, so
// that the partials of a long cache are read at once rather than one after the other
template <int HD, int MODE>
__device__ __forceinline__ void a8_merge_one(const A8& A, int cw, const int bx, const int seq, float (&sum)[1024 / HD][HD]) {
    constexpr int NG = 1024 / HD;  // chunk groups
    const int tid = threadIdx.x, lane = tid & 63, d = 4 * (tid % (HD / 4)), grp = tid / (HD / 4);
    const int h = bx % A.nkv, x = bx / A.nkv;
    const int cb = x / cw, cc = x % cw;
    int beg, end;
    a8_tiles(A, a8_len(A, seq), cb * cw, cw, beg, end);
    const int live = max(1, (end - beg + A.tpc - 1) / A.tpc);
    const int64_t step = (int64_t)cw * (HD + 2);
    const float* part = A.ws + (int64_t)((seq * A.nkv + h) * A.ncb + cb) * A.chunks * step;
    const float* st = part + cw * HD + 2 * cc;
    const float* val = part + cc * HD + d;
    float M = -INFINITY, L = 0.0f;
    for (int k = lane; k < live; k += 64) M = fmaxf(M, st[k * step]);
    M = aeth_wave_max(M);
    for (int k = lane; k < live; k += 64) {
        const float2 ml = *(const float2*)(st + k * step);
        L += (ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M)) * ml.y;
    }
    L = aeth_wave_sum(L);
    a8_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = grp; k < live; k += NG) {
        const float m = st[k * step];
        acc += *(const a8_f4*)(val + k * step) * (m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M));
    }
    *(a8_f4*)&sum[grp][d] = acc;
    if constexpr ((MODE & A8_STAT) != 0)
        if (tid == 0) *(float2*)(A.stat + 2 * ((int64_t)(seq * A.nkv + h) * A.cols + x)) = make_float2(M, 1.0f / L);
    __syncthreads();
    if (tid >= HD) return;
    float y = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; g++) y += sum[g][tid];
    A.out[((int64_t)seq * A.n + x / A.G) * ((int64_t)A.nq * HD) + (int64_t)(h * A.G + x % A.G) * HD + tid] = L == 0.0f ? 0.0f : y * (1.0f / L);
}

template <int HD, int MODE>
__global__ void __launch_bounds__(256) k_attn8_merge(A8 A, int cw) {
    __shared__ __attribute__((aligned(16))) float sum[1024 / HD][HD];
    a8_merge_one<HD, MODE>(A, cw, blockIdx.x, blockIdx.y, sum);
}

// The same for at most 8 chunks: hd / 4 lanes a column, its partials all in flight at once
template <int HD, int MODE>
__device__ __forceinline__ void a8_merge_some(const A8& A, int cw, const int bx, const int seq) {
    constexpr int MOST = 8;
    const int unit = (bx * 256 + threadIdx.x) / (HD / 4), d = 4 * (threadIdx.x % (HD / 4));
    if (unit >= A.nkv * A.cols) return;
    const int h = unit / A.cols, x = unit % A.cols, cb = x / cw, cc = x % cw;
    int beg, end;
    a8_tiles(A, a8_len(A, seq), cb * cw, cw, beg, end);
    const int live = max(1, (end - beg + A.tpc - 1) / A.tpc);
    const int64_t step = (int64_t)cw * (HD + 2);
    const float* part = A.ws + (int64_t)((seq * A.nkv + h) * A.ncb + cb) * A.chunks * step;
    float2 ml[MOST];
    a8_f4 v[MOST];
#pragma unroll
    for (int k = 0; k < MOST; k++)
        if (k < A.chunks) {  // (uniform)
            const int64_t at = min(k, live - 1) * step;
            ml[k] = *(const float2*)(part + at + cw * HD + 2 * cc);
            v[k] = *(const a8_f4*)(part + at + cc * HD + d);
        }
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int k = 0; k < MOST; k++)
        if (k < A.chunks) M = fmaxf(M, ml[k].x);
    a8_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < MOST; k++)
        if (k < A.chunks) {
            const float w = ml[k].x == -INFINITY || k >= live ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - M);
            const bool in = k < live;
            L += in ? w * ml[k].y : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += in ? v[k][e] * w : 0.0f;
        }
    if constexpr ((MODE & A8_STAT) != 0)
        if (d == 0) *(float2*)(A.stat + 2 * ((int64_t)(seq * A.nkv + h) * A.cols + x)) = make_float2(M, 1.0f / L);
    acc = L == 0.0f ? (a8_f4){0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / L);
    float* dst = A.out + ((int64_t)seq * A.n + x / A.G) * ((int64_t)A.nq * HD) + (int64_t)(h * A.G + x % A.G) * HD + d;
    if (A.ovec) *(a8_f4*)dst = acc;
    else dst[0] = acc[0], dst[1] = acc[1], dst[2] = acc[2], dst[3] = acc[3];
}

template <int HD, int MODE>
__global__ void __launch_bounds__(256) k_attn8_merge_few(A8 A, int cw) { a8_merge_some<HD, MODE>(A, cw, blockIdx.x, blockIdx.y); }

// A workgroup a column costs a µs for each thousand of them (16000 columns in 2 chunks: 25 µs, 9 with 32 lanes each; 8000 in 8:
// 15 and 8); of a few columns it has more of many chunks in flight (256 columns in 8 chunks: 0.8 µs less, 1024: 0.2).
inline bool a8_merge_is_some(const A8& A, int64_t seqs) {
    return A.chunks <= 4 || (A.chunks <= 8 && (int64_t)A.nkv * A.cols * seqs >= 6 * (int64_t)aeth_num_cus());
}
template <int HD, int MODE>
void a8_merge(const A8& A, int cw, int64_t seqs, hipStream_t s) {
    const int64_t cols = (int64_t)A.nkv * A.cols;
    if (a8_merge_is_some(A, seqs))
        hipLaunchKernelGGL((k_attn8_merge_few<HD, MODE>), dim3((unsigned)aeth_cdiv(cols * (HD / 4), 256), (unsigned)seqs), dim3(256), 0, s, A, cw);
    else hipLaunchKernelGGL((k_attn8_merge<HD, MODE>), dim3((unsigned)cols, (unsigned)seqs), dim3(256), 0, s, A, cw);
}

// The form a call takes: the columns of a workgroup and, where its column blocks are fewer than `target`, the chunks of at
// least tiles_min tiles that they are split into.
struct Form {
    int cw, chunks, tpc;
};
Form a8_split(int cw, int64_t units, int64_t span, int64_t target, int64_t tiles_min) {
    const int64_t want = std::max<int64_t>(1, std::min(aeth_cdiv(target, units), aeth_cdiv(span, tiles_min)));
    const int64_t tpc = std::max<int64_t>(4, aeth_cdiv(aeth_cdiv(span, want), 4) * 4);
    return {cw, (int)std::max<int64_t>(1, aeth_cdiv(span, tpc)), (int)tpc};
}
// tiles a block of cw columns sees at most: a window's, or all of max_len
int64_t a8_span(int64_t cw, int64_t n, int64_t G, int64_t max_len, int64_t window) {
    const int64_t all = aeth_cdiv(max_len, KV8_TILE), rows = std::min(aeth_cdiv(cw, G) + 1, n);
    return window > 0 ? std::min(all, (window + rows + 62) / KV8_TILE + 1) : all;
}
// (column blocks of cw) x (tiles each sees), over one head
double a8_blocks_tiles(int64_t cw, int64_t cols, int64_t n, int64_t G, int64_t max_len, int64_t window) {
    const double blocks = (double)aeth_cdiv(cols, cw), most = (double)a8_span(cw, n, G, max_len, window);
    if (window > 0) return blocks * most;
    return blocks * ((double)max_len - 0.5 * (double)n) / KV8_TILE + 0.5 * blocks;
}
Form a8_form(int64_t seqs, int64_t n, int64_t G, int64_t nkv, int64_t hd, int64_t max_len, int64_t window, bool ragged) {
    const int64_t cus = aeth_num_cus(), cols = n * G, heads = seqs * nkv;
    auto span = [&](int64_t cw) { return a8_span(cw, n, G, max_len, window); };
    auto units = [&](int64_t cw) { return heads * aeth_cdiv(cols, cw); };
    // 16 columns: split until two workgroups a CU have work; four, where the device alone knows the length, so that one below it has
    // work for more (a decode step's layer of a small model, its products included, one / two / four a CU: 4000 tokens in a cache of
    // their size 26.6 / 26.7 / 26.6 µs, 8000 28.8 / 27.0 / 27.0, 131000 72.5 / 73.1 / 79.0); not up to 512 tokens, two tiles a wave (a token over
    // 300: 7.8 µs, 8.4 in two chunks; over 600: 9.7, 8.9 in three)
    const Form small = a8_split(16, units(16), span(16), span(16) <= 8 ? 1 : (ragged ? 4 : 2) * cus, 4);
    if (ragged && seqs > 1) {
        // A batch: the least, in µs, of 5 + ((0.34·tpc)^1.5 + max(MB / 6.4, 1.5·r)^1.5)^(2/3) + 0.2·wgs/CU, and where it is split 2.2 +
        // 0.19 for each 100,000 floats of partials: tpc the longest workgroup's tiles, MB what is read if lengths are spread
        // evenly up to max_len, r the rounds of workgroups (three on a CU at once). 32 / 8 heads of 128, measured and (as reckoned)
        // whole / in two / in four chunks: 64 sequences of up to 300 tokens 10 (10) / 13 (13), 1000 18 (19) / 22 (21), 4096 56 (58) / 55 (56) /
        // 52 (56); 24 of up to 4096 31 (34) / 32 (29) / 29 (27), 8 29 (29) / 21 (20) / 16 (16).
        const double sp = (double)span(16), f4 = hd == 64 ? 0.5 : hd == 128 ? 1.0 : 2.0;
        const double mb = (double)units(16) * (window > 0 ? sp : 0.5 * sp + 0.5) * (double)aeth_kv8_tile_bytes((int)hd) * 1e-6;
        Form best = small;
        double least = INFINITY;
        for (int64_t target : {(int64_t)1, cus, 2 * cus, 4 * cus}) {
            const Form f = a8_split(16, units(16), span(16), target, 4);
            const double wgs = (double)(units(16) * f.chunks) / (double)cus, rounds = std::ceil(std::ceil(wgs) / (hd == 64 ? 4.0 : 3.0));
            const double chain = 0.34 * f4 * std::min((double)f.tpc, sp), flow = std::max(mb / 6.4, 1.5 * f4 * rounds);
            double t = 5.0 + std::cbrt(std::pow(chain * std::sqrt(chain) + flow * std::sqrt(flow), 2.0)) + 0.2 * f4 * wgs;
            if (f.chunks > 1) t += 2.2 + 1.9e-6 * (double)(heads * cols * f.chunks) * (double)(hd + 2);
            if (t < least) {
                least = t;
                best = f;
            }
        }
        return best;
    }
    // Up to 64 columns half of the smallest of the other forms has none (64 columns over 1000 / 5000 / 30000 tokens: 10.0 / 15.4 /
    // 34.6 µs, with 128 columns 26 / 27 / 42 at best; at head_dim 64 7.7 / 10.7 / 22.2, 19 / 20 / 30). A call whose length the device
    // alone knows has at most 64 (one query a sequence) but for more query heads a KV head than that; head_dim 256 has no other
    // form (4 query heads each: a 512-token prompt 46 µs, 2000 tokens 301, a token over 30000 34).
    if (hd > 128 || cols <= 64 || ragged) return small;
    // Otherwise the least of what the forms take, in µs on a CU's share of the tiles (w; q: the fullest CU's of few workgroups),
    // its workgroups' rounds (r: three at once, four) and the tiles of one (tpc), at head_dim 128 (64):
    //   16 columns  max(5.5 + 0.45·tpc, 6 + 0.33·q + 4.5·r) (5 + 0.3·tpc, 5 + 0.185·q + 2.8·r)
    //   128         max(8 + 2.3·tpc, 22 + 1.96·w) (7 + 1.53·tpc, 15 + 1.25·w): two workgroups a CU
    //   256         12 + 2.8·max(tpc, w) + 1.5·max(0, w - 0.4·max(tpc, w)): one a CU, whose codes serve twice the columns; the chip
    //               clocks lower when it is full
    //   a split's join: 3, and one for each 4 MB of partials (16 columns: 2.5, 2 MB).
    // 8 KV heads of 128, measured and (as reckoned) with 16 / 128 / 256 columns: 4 query heads each, 1000 tokens 40 (41) / 43 (44) /
    // 56 (56), 2000 110 (116) / 86 (84) / 104 (101), 4000 375 (383) / 265 (265) / 252 (245), 1000 queries over 6000 in one / two /
    // two chunks 248 (247) / 206 (202) / 194 (194), 70 over 30000 with 16 columns in 2, 4 and 8 chunks 169 (169), 130 (131), 114 (119);
    // 2 query heads each, 2000 tokens 59 (61) / 74 (80) / 100 (100); one each, 512 tokens 10 (12), in two chunks 14 (17).
    // At head_dim 64, 4 query heads each: 2000 tokens 60 (63) / 56 (55), 250 queries over 20000 127 (123), in 8 chunks of 128 112 (120).
    const double c = (double)cus;
    Form best = small;
    double least = INFINITY;
    for (int64_t cw = 16; cw <= (hd == 128 ? 256 : 128); cw = std::max<int64_t>(128, 2 * cw)) {
        const double tiles = (double)heads * a8_blocks_tiles(cw, cols, n, G, max_len, window);
        for (int64_t target : {(int64_t)0, cus, 2 * cus, 4 * cus}) {  // workgroups split for
            if (target > (cw == 16 ? 4 : cw == 128 ? 2 : 1) * cus) continue;
            const Form f = a8_split(cw, units(cw), span(cw), std::max<int64_t>(1, target), cw == 16 ? 4 : 8);
            const int64_t wgs = units(cw) * f.chunks;
            const double w = tiles / c, tpc = (double)std::min<int64_t>(f.tpc, span(cw));
            const double u = (double)aeth_cdiv(wgs, cus), q = u * (tiles / (double)wgs);
            const double own = std::max(tpc, w);
            double t = cw == 256   ? 12.0 + 2.8 * own + 1.5 * std::max(0.0, w - 0.4 * own)
                       : cw == 128 ? (hd == 128 ? std::max(8.0 + 2.3 * tpc, 22.0 + 1.96 * w) : std::max(7.0 + 1.53 * tpc, 15.0 + 1.25 * w))
                       : hd == 128 ? std::max(5.5 + 0.45 * tpc, 6.0 + 0.33 * q + 4.5 * std::ceil(u / 3.0))
                                   : std::max(5.0 + 0.3 * tpc, 5.0 + 0.185 * q + 2.8 * std::ceil(u / 4.0));
            if (f.chunks > 1) t += (cw == 16 ? 2.5 : 3.0) + (cw == 16 ? 2e-6 : 1e-6) * (double)(heads * cols * f.chunks) * (double)(hd + 2);
            if (t < least) {
                least = t;
                best = f;
            }
        }
    }
    return best;
}

template <int HD, int MODE>
int a8_launch(const A8& A, const Form& f, int64_t seqs, hipStream_t s) {
    const dim3 grid((unsigned)((int64_t)A.nkv * A.ncb), (unsigned)seqs, (unsigned)A.chunks);
    if (f.cw == 16) hipLaunchKernelGGL((k_attn8<HD, MODE>), grid, dim3(256), 0, s, A);
    if constexpr (HD <= 128)
        if (f.cw == 128) hipLaunchKernelGGL((k_attn8p<HD, 4, MODE>), grid, dim3(256), 0, s, A);
    if constexpr (HD == 128)
        if (f.cw == 256) hipLaunchKernelGGL((k_attn8p<HD, 8, MODE>), grid, dim3(512), 0, s, A);
    AETH_LAUNCH_CHECK();
    if constexpr ((MODE & A8_PART) == 0) {
        if (A.chunks > 1) {
            a8_merge<HD, MODE>(A, f.cw, seqs, s);
            AETH_LAUNCH_CHECK();
        }
    }
    return AETH_OK;
}

// A call's arguments for its form
inline A8 a8_args(const float* q, int64_t q_stride, const void* cache, int64_t seq_bytes, const int* lens, int len_add, int64_t n, int64_t nq, int64_t nkv,
                  int64_t max_seq, int64_t max_len, int64_t window, float* out, void* ws) {
    A8 A = {};
    A.q = q;
    A.q_stride = q_stride;
    A.cache = (const uint8_t*)cache;
    A.seq_bytes = seq_bytes;
    A.lens = lens;
    A.len_add = len_add;
    A.max_len = (int)max_len;
    A.n = (int)n;
    A.nq = (int)nq;
    A.nkv = (int)nkv;
    A.G = (int)(nq / nkv);
    A.cols = (int)(n * A.G);
    A.tiles = (int)aeth_cdiv(max_seq, KV8_TILE);
    A.window = window > 0 && window < max_len ? (int)window : 0;  // one that reaches past key 0 masks nothing
    A.out = out;
    A.ws = (float*)ws;
    A.qvec = ((uintptr_t)q & 15) == 0 && (q_stride & 3) == 0;
    A.ovec = ((uintptr_t)out & 15) == 0;
    return A;
}
inline void a8_take(A8& A, const Form& f) {
    A.ncb = (int)aeth_cdiv(A.cols, f.cw);
    A.tpc = f.tpc;
    A.chunks = f.chunks;
}

}  // namespace
