// Attention over the 8-bit cache in two further forms (the mathematics and kernels of the attention itself: aeth_attn_kv8_dev.hpp).
//
// A shared prefix. The rows of a batch stand behind the same first P tokens, held once. The softmax over a row's
// keys is a sum over parts: with m_j, l_j, o_j the maximum, sum and weighted values of part j, M = max m_j,
//   out = Σ_j 2^(m_j - M) o_j / Σ_j 2^(m_j - M) l_j.
// So the prefix is one product of all rows of a KV head, n_seqs·G columns, with no order among them, and reads its keys once
// for as many columns as a workgroup holds; each sequence's own tokens are the batch's attention; both leave
// their parts in the workspace and k_attn8_join joins them.
//
// The weights that tokens receive. weights[t] = prior[t] + Σ_x 2^(s_x(t) - m_x) / l_x over the columns x that see t. m_x and l_x are
// known behind the attention. Of few columns (SCORES) its workgroups also leave their scores, 4 bytes a column and key where a
// key's codes are 2·hd + 8 (k_kv8_weigh_scores); of more the scores are formed once more from the keys (k_kv8_weigh), where they are summed
// over columns in registers: no score reaches memory. Every sum has a fixed order.
#include "aeth_attn_kv8_dev.hpp"

namespace {

// ── a shared prefix ───────────────────────────────────────────────────────

// Both attentions in one launch, each a share of the workgroups: the prefix's products keep the matrix units busy, the sequences' own
// tokens the memory. The first `prefixes` workgroups take the prefix in columns of cw (16, or 128 in the form for many), the others a sequence
// each (its chunks after one another: the first ones, which every sequence has, first). 32 / 8 heads of 128: 2 sequences behind 1000 tokens
// 7.1 µs (in two launches 6.8 and 5.7), 160 of up to 500 tokens behind 20000 125 (138 and 25): what bounds that is the prefix's products, 0.42
// PFLOP/s of the formula, 0.84 of the matrix units', as in aeth_attn_kv8's long prompts. 160 copies of the prefix in a batch's own caches take 1101.
template <int HD, int CW>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_attn8_shared(A8 P, A8 O, int prefixes, int seqs) {
    constexpr int MAX = CW == 128 ? std::max((int)sizeof(float[4][16][HD + 4]), 2 * (HD / 8) * A8_KF) : (int)sizeof(float[4][16][HD + 4]);
    __shared__ __attribute__((aligned(16))) char lds[MAX];
    __shared__ float pm[4][16], pl[4][16];
    uint32_t(&none)[2][HD / 4] = *(uint32_t(*)[2][HD / 4])lds;  // a decode step's, which no form here has
    float(&po)[4][16][HD + 4] = *(float(*)[4][16][HD + 4])lds;
    const int bx = blockIdx.x;
    if (bx >= prefixes) {
        const int per = O.nkv * O.ncb, at = bx - prefixes, unit = at / per;
        a8_few<HD, A8_PART>(O, at % per, unit % seqs, unit / seqs, po, pm, pl, none);
    } else if constexpr (CW == 128) {
        __shared__ __attribute__((aligned(16))) char vb[2][HD * 128];
        __shared__ __attribute__((aligned(16))) float sc[2][2 * KV8_TILE];
        const int per = P.nkv * P.ncb;
        a8_many<HD, 4, A8_FLAT | A8_PART>(P, bx % per, 0, bx / per, *(char(*)[2][HD / 8 * A8_KF])lds, vb, sc);
    } else {
        const int per = P.nkv * P.ncb;
        a8_few<HD, A8_FLAT | A8_PART>(P, bx % per, 0, bx / per, po, pm, pl, none);
    }
}

// A column's parts: of the prefix (P, in blocks of cw columns), then of its own tokens (O, of 16). Part k: its maximum and sum, its value from dimension d on
template <int HD>
struct Parts {
    const float *p, *o;
    int64_t step_p, step_o;
    int of_p, stat_p, value_p, stat_o, value_o;  // parts of the prefix; offsets in a part
    __device__ __forceinline__ Parts(const A8& P, int cw, const A8& O, int seq, int unit, int d) {
        const int h = unit / O.G, g = unit % O.G, x = seq * O.G + g;
        step_p = (int64_t)cw * (HD + 2);
        step_o = 16 * (HD + 2);
        p = P.ws + (int64_t)(h * P.ncb + x / cw) * P.chunks * step_p;
        o = O.ws + (int64_t)((seq * O.nkv + h) * O.ncb + g / 16) * O.chunks * step_o;
        of_p = P.chunks;
        stat_p = cw * HD + 2 * (x % cw);
        value_p = x % cw * HD + d;
        stat_o = 16 * HD + 2 * (g % 16);
        value_o = g % 16 * HD + d;
    }
    __device__ __forceinline__ float2 stat(int k) const { return *(const float2*)(k < of_p ? p + k * step_p + stat_p : o + (k - of_p) * step_o + stat_o); }
    __device__ __forceinline__ a8_f4 value(int k) const { return *(const a8_f4*)(k < of_p ? p + k * step_p + value_p : o + (k - of_p) * step_o + value_o); }
};
// parts with something in them: all of the prefix's, the first of a sequence's own
__device__ __forceinline__ int sv_live(const A8& P, const A8& O, int seq, int g) {
    int beg, end;
    a8_tiles(O, a8_len(O, seq), g / 16 * 16, 16, beg, end);
    return P.chunks + max(1, (end - beg + O.tpc - 1) / O.tpc);
}

// Joins many parts (2 sequences behind 60000 tokens, 60 parts): a workgroup a column, HD/4 lanes of four dimensions for every 1024/HD-th part
template <int HD>
__global__ void __launch_bounds__(256) k_attn8_join(A8 P, int cw, A8 O) {
    constexpr int L = HD / 4, GR = 256 / L;
    __shared__ __attribute__((aligned(16))) float sum[GR][HD];
    const int tid = threadIdx.x, lane = tid & 63, d = 4 * (tid % L), grp = tid / L, seq = blockIdx.y, unit = blockIdx.x;
    const int live = sv_live(P, O, seq, unit % O.G);
    const Parts<HD> part(P, cw, O, seq, unit, d);
    float M = -INFINITY, S = 0.0f;
    for (int k = lane; k < live; k += 64) M = fmaxf(M, part.stat(k).x);
    M = aeth_wave_max(M);
    for (int k = lane; k < live; k += 64) {
        const float2 ml = part.stat(k);
        S += (ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M)) * ml.y;
    }
    S = aeth_wave_sum(S);
    a8_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = grp; k < live; k += GR) {
        const float m = part.stat(k).x;
        acc += part.value(k) * (m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - M));
    }
    *(a8_f4*)&sum[grp][d] = acc;
    __syncthreads();
    if (tid >= HD) return;
    float y = 0.0f;
#pragma unroll
    for (int i = 0; i < GR; i++) y += sum[i][tid];
    O.out[(int64_t)seq * ((int64_t)O.nq * HD) + (int64_t)unit * HD + tid] = S == 0.0f ? 0.0f : y * (1.0f / S);
}

// ... and at most MOST, 8 or 16: HD/4 lanes a column, its parts all in flight at once, those without content too (they are left out behind the length,
// which is still on its way: 2 sequences of 32 heads 3.4 µs, 5.0 where their number was waited for; 160 of 13 parts 8.8, 13.1 with a workgroup a
// column)
constexpr int JOIN_FEW = 8, JOIN_MORE = 16;
template <int HD, int MOST>
__global__ void __launch_bounds__(256) k_attn8_join_few(A8 P, int cw, A8 O) {
    constexpr int L = HD / 4;
    const int unit = (blockIdx.x * 256 + threadIdx.x) / L, d = 4 * (threadIdx.x % L), seq = blockIdx.y, all = P.chunks + O.chunks;
    if (unit >= O.nkv * O.G) return;
    const Parts<HD> part(P, cw, O, seq, unit, d);
    float2 ml[MOST];
    a8_f4 v[MOST];
#pragma unroll
    for (int k = 0; k < MOST; k++)
        if (k < all) {  // (uniform)
            ml[k] = part.stat(k);
            v[k] = part.value(k);
        }
    const int live = sv_live(P, O, seq, unit % O.G);
    float M = -INFINITY, S = 0.0f;
#pragma unroll
    for (int k = 0; k < MOST; k++)
        if (k < all) M = k < live ? fmaxf(M, ml[k].x) : M;
    a8_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < MOST; k++)
        if (k < all) {
            // (a part whose visible scores are all NaN has the maximum -Inf and the sum NaN, and 0·NaN keeps it; one that sees nothing adds 0·0)
            const bool in = k < live;
            const float w = ml[k].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[k].x - M);
            S += in ? w * ml[k].y : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] += in ? v[k][e] * w : 0.0f;
        }
    acc = S == 0.0f ? (a8_f4){0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / S);
    float* dst = O.out + (int64_t)seq * ((int64_t)O.nq * HD) + (int64_t)unit * HD + d;
    if (O.ovec) *(a8_f4*)dst = acc;
    else dst[0] = acc[0], dst[1] = acc[1], dst[2] = acc[2], dst[3] = acc[3];
}

// The prefix's form, 16 or 128 columns: a8_form's reckoning for columns that all see `span` tiles, `own` chunks of the sequences' own tokens beside
// them; chunks of 128 columns take any length, as even as they can be, and what a part-filled round adds is counted by half. 32 / 8 heads of 128, µs
// with the form taken (the best of 10 to 13 tried): 1000 sequences behind 2000 tokens 175, 128 columns in 1 chunk (175); 256 behind 6000 86, 128 in 4
// (84); 200 behind 12000 117, 128 in 4 (113, 8); 160 behind 10000 78, 128 in 6 (78); 160 behind 20000 132, 128 in 12 (130; 6 chunks 137, 7 162);
// 120 behind 20000 111, 128 in 8 (111); 64 behind 3000 21.5, 16 in 2 (21.5); 48 behind 4001 32, 16 in 2 (29, 4); 32 behind 8000 22.3, 16 in 4 (22.3);
// 17 behind 20000 32, 16 in 6 (32). The 256-column form, whose workgroup fills a CU, has no room for the sequences' own beside it.
Form sv_prefix_form(int64_t cols, int64_t nkv, int64_t hd, int64_t span, int64_t own) {
    const int64_t cus = aeth_num_cus();
    // (at head_dim 256 a workgroup fills a CU: 32 sequences behind 8000 tokens of 16 / 4 heads in 8 chunks 33 µs, in 16 41)
    const Form small = a8_split(16, nkv * aeth_cdiv(cols, 16), span, (hd == 256 ? 1 : 2) * cus, 4);
    if (hd > 128 || cols <= 64) return small;
    const double c = (double)cus;
    Form best = small;
    double least = INFINITY;
    for (int64_t cw : {16, 128}) {
        const int64_t units = nkv * aeth_cdiv(cols, cw);
        const double tiles = (double)units * (double)span;
        const int64_t limit = (cw == 16 ? 4 : 2) * cus;
        for (int64_t target : {(int64_t)0, cus, 2 * cus, limit, cus / units * units, (cw == 128 ? 2 * cus / units * units : cus),
                               std::min(limit, units * std::max<int64_t>(1, JOIN_FEW - own))}) {
            Form f = a8_split(cw, units, span, std::max<int64_t>(1, target), cw == 16 ? 4 : 8);
            if (cw == 128) {
                f.tpc = (int)aeth_cdiv(span, f.chunks);
                f.chunks = (int)aeth_cdiv(span, f.tpc);
            }
            const int64_t wgs = units * f.chunks;
            const double w = tiles / c, tpc = (double)std::min<int64_t>(f.tpc, span);
            const double u = (double)aeth_cdiv(wgs, cus), q = u * (tiles / (double)wgs);
            double t = cw == 128   ? (hd == 128 ? std::max(8.0 + 2.3 * tpc, 22.0 + 0.98 * (w + q)) : std::max(7.0 + 1.53 * tpc, 15.0 + 0.625 * (w + q)))
                       : hd == 128 ? std::max(5.5 + 0.45 * tpc, 6.0 + 0.33 * q + 4.5 * std::ceil(u / 3.0))
                                   : std::max(5.0 + 0.3 * tpc, 5.0 + 0.185 * q + 2.8 * std::ceil(u / 4.0));
            t += (cw == 128 && hd == 128 ? 1.5e-6 : 3e-6) * (double)(nkv * cols * f.chunks) * (double)(hd + 2);
            if (f.chunks + own > (cw == 128 ? JOIN_MORE : JOIN_FEW)) t += 2.5;
            if (t < least) {
                least = t;
                best = f;
            }
        }
    }
    return best;
}

// bytes of the parts: no more than target + units blocks of columns in any form (a8_split)
int64_t sv_prefix_ws(int64_t seqs, int64_t nq, int64_t nkv, int64_t hd) {
    const int64_t cols = seqs * (nq / nkv), cus = aeth_num_cus();
    auto need = [&](int64_t cw, int64_t target) { return (target + nkv * aeth_cdiv(cols, cw)) * cw; };
    int64_t most = need(16, 4 * cus);
    if (hd <= 128 && cols > 64) most = std::max(most, need(128, 2 * cus));
    return most * (hd + 2) * (int64_t)sizeof(float);
}
int64_t sv_own_ws(int64_t seqs, int64_t nq, int64_t nkv, int64_t hd) {
    return (4 * aeth_num_cus() + seqs * nkv * aeth_cdiv(nq / nkv, 16)) * 16 * (hd + 2) * (int64_t)sizeof(float);
}

template <int HD>
int sv_shared(A8 P, A8 O, int64_t seqs, hipStream_t s) {
    const Form fo = a8_form(seqs, 1, O.G, O.nkv, HD, O.max_len, O.window, true);
    a8_take(O, fo);
    Form fp = {16, 0, 4};
    if (P.max_len > 0) {
        const int64_t span = aeth_cdiv(P.max_len, KV8_TILE) - (P.window > 0 ? std::max(0, P.max_len - P.window) / KV8_TILE : 0);
        fp = sv_prefix_form(P.cols, P.nkv, HD, span, O.chunks);
    }
    a8_take(P, fp);
    const int64_t prefixes = (int64_t)P.nkv * P.ncb * P.chunks, own = (int64_t)O.nkv * O.ncb * seqs * O.chunks;
    const dim3 grid((unsigned)(prefixes + own)), block(256);
    if (fp.cw == 16) hipLaunchKernelGGL((k_attn8_shared<HD, 16>), grid, block, 0, s, P, O, (int)prefixes, (int)seqs);
    if constexpr (HD <= 128)
        if (fp.cw == 128) hipLaunchKernelGGL((k_attn8_shared<HD, 128>), grid, block, 0, s, P, O, (int)prefixes, (int)seqs);
    AETH_LAUNCH_CHECK();
    const int64_t cols = (int64_t)O.nkv * O.G;
    const int parts = P.chunks + O.chunks;
    const dim3 few((unsigned)aeth_cdiv(cols, 1024 / HD), (unsigned)seqs);
    if (parts <= JOIN_FEW) hipLaunchKernelGGL((k_attn8_join_few<HD, JOIN_FEW>), few, block, 0, s, P, fp.cw, O);
    else if (parts <= JOIN_MORE) hipLaunchKernelGGL((k_attn8_join_few<HD, JOIN_MORE>), few, block, 0, s, P, fp.cw, O);
    else hipLaunchKernelGGL(k_attn8_join<HD>, dim3((unsigned)cols, (unsigned)seqs), block, 0, s, P, fp.cw, O);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

// ── the weights that tokens receive ───────────────────────────────────────

struct Weigh {
    const float* prior;  // [seqs][nkv][max_seq]; nullptr: zeros
    float* weights;
    int64_t max_seq;
    float* part;         // k_kv8_weigh in several chunks of columns: [chunks][nkv][keys]
    int chunks, per;     // of `per` blocks of columns, as many as the keys' columns have
    int first, full;     // the first group of keys that some column sees; so many from there have all chunks
    int64_t keys;        // of a row of part, from that group on: whole groups
    int wgs;             // workgroups a head
};

// The maximum and 1 / sum of a column: as the attention left it, or from its chunks' parts (every lane of the wave calls it, and
// every lane has the result)
template <int HD>
__device__ __forceinline__ float2 sv_column(const A8& A, int len, int seq, int h, int x) {
    const int64_t unit = (int64_t)seq * A.nkv + h;
    if (A.chunks == 1) return *(const float2*)(A.stat + 2 * (unit * A.cols + x));
    int beg, end;
    a8_tiles(A, len, x / 16 * 16, 16, beg, end);
    const int live = max(1, (end - beg + A.tpc - 1) / A.tpc), lane = threadIdx.x & 63;
    const int64_t step = 16 * (HD + 2);
    const float* st = A.ws + (unit * A.ncb + x / 16) * A.chunks * step + 16 * HD + 2 * (x % 16);
    // (a part whose visible scores are all NaN has the maximum -Inf and the sum NaN: 0·NaN keeps it)
    auto weight = [](float x, float m) { return x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - m); };
    float2 ml = make_float2(-INFINITY, 0.0f);
    for (int k = lane; k < live; k += 64) {
        const float2 more = *(const float2*)(st + k * step);
        const float m = fmaxf(ml.x, more.x);
        ml.y = ml.y * weight(ml.x, m) + more.y * weight(more.x, m);
        ml.x = m;
    }
    const float M = aeth_wave_max(ml.x);
    const float S = aeth_wave_sum(ml.y * weight(ml.x, M));
    return make_float2(M, 1.0f / S);
}

// From the scores: workgroup (256·KT keys, KV head), the columns 32 at a time, their statistics first. Latency bounds it: a length, chunks'
// statistics, the sum.
template <int HD, int KT>
__device__ __forceinline__ void sv_weigh_scores(const A8& A, const Weigh& W, int bx, int seq, float2 (&col)[32]) {
    const int tid = threadIdx.x, h = bx % A.nkv, t0 = bx / A.nkv * (256 * KT);
    const int len = a8_len(A, seq);
    if (t0 >= len) return;  // (uniform)
    const int64_t unit = (int64_t)seq * A.nkv + h, row = 64 * (int64_t)A.score_tiles;
    const float* src = A.scores + unit * A.cols * row;
    int t[KT];
#pragma unroll
    for (int k = 0; k < KT; k++) t[k] = t0 + tid + 256 * k;
    float s[4][KT];  // four columns' scores, asked for before what their sums wait for
    auto fetch = [&](int x) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int k = 0; k < KT; k++) s[j][k] = src[min(x + j, A.cols - 1) * row + min(t[k], (int)row - 1)];
    };
    fetch(0);
    float prior[KT], sum[KT];
#pragma unroll
    for (int k = 0; k < KT; k++) {
        prior[k] = t[k] < len && W.prior ? W.prior[unit * W.max_seq + t[k]] : 0.0f;
        sum[k] = 0.0f;
    }
    for (int c0 = 0; c0 < A.cols; c0 += 32) {
        const int count = min(32, A.cols - c0);
        if (c0 > 0) __syncthreads();
        for (int c = tid >> 6; c < count; c += 4) {
            const float2 ml = sv_column<HD>(A, len, seq, h, c0 + c);
            if ((tid & 63) == 0) col[c] = ml;
        }
        __syncthreads();
        const int hi0 = len - A.n + 1;
        for (int c1 = 0; c1 < count; c1 += 4) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int x = c0 + c1 + j, hi = A.n > 1 ? hi0 + x / A.G : hi0, lo = A.window > 0 ? hi - A.window : 0;  // (uniform)
                const float2 ml = col[min(c1 + j, 31)];
#pragma unroll
                for (int k = 0; k < KT; k++)
                    if (x < A.cols && t[k] >= lo && t[k] < hi) sum[k] = fmaf(__builtin_amdgcn_exp2f(s[j][k] - ml.x), ml.y, sum[k]);
            }
            if (c0 + c1 + 4 < A.cols) fetch(c0 + c1 + 4);
        }
    }
#pragma unroll
    for (int k = 0; k < KT; k++)
        if (t[k] < len) W.weights[unit * W.max_seq + t[k]] = prior[k] + sum[k];
}

template <int HD, int KT>
__global__ void __launch_bounds__(256) k_kv8_weigh_scores(A8 A, Weigh W) {
    __shared__ float2 col[32];
    sv_weigh_scores<HD, KT>(A, W, blockIdx.x, blockIdx.y, col);
}

// The join of the attention's chunks (the first `joins` workgroups) and the weights, which only share what they read, in one launch. 32 / 8
// heads: a token over 2049 3.5 µs (a launch each: 3.3 and 7.8), 32 sequences of up to 4096 7.5 (4.6 and 10.1; 9.1 with one key a thread).
template <int HD, bool SOME, int KT>
__global__ void __launch_bounds__(256) k_kv8_join_weigh(A8 A, Weigh W, int joins) {
    __shared__ __attribute__((aligned(16))) float sum[1024 / HD][HD];
    __shared__ float2 col[32];
    const int bx = blockIdx.x;
    if (bx >= joins) sv_weigh_scores<HD, KT>(A, W, bx - joins, blockIdx.y, col);
    else if constexpr (SOME) a8_merge_some<HD, 0>(A, 16, bx, blockIdx.y);
    else a8_merge_one<HD, 0>(A, 16, bx, blockIdx.y, sum);
}

// Keys of a workgroup of k_kv8_weigh: two halves of 32 a wave, or one where a half's codes take as many registers
constexpr int sv_group(int hd) { return hd == 256 ? 256 : 512; }

// The blocks of 32 columns that see a key of k0 .. k0 + keys - 1: from column x_beg on
struct Seen {
    int x_beg, x_end, blocks;
};
__host__ __device__ inline Seen sv_seen(int n, int G, int len, int window, int64_t k0, int keys) {
    const int past = len - n;  // keys before the first query
    const int64_t i0 = k0 > past ? k0 - past : 0;
    int64_t i1 = n;
    if (window > 0) {
        const int64_t last = (k0 + keys < len ? k0 + keys : len) - 1 + (int64_t)window - past;
        i1 = last < i1 ? last : i1;
    }
    if (i1 <= i0) return {0, 0, 0};
    return {(int)(i0 * G), (int)(i1 * G), (int)(((i1 - i0) * G + 31) / 32)};
}

// The chunks of a group's columns
__device__ __forceinline__ int sv_count(const A8& A, const Weigh& W, int group, int gk) {
    return max(1, (sv_seen(A.n, A.G, A.max_len, A.window, gk * (int64_t)group, gk).blocks + W.per - 1) / W.per);
}

// Many columns: a wave keeps NT·32 keys as fp16 in registers, its workgroup of eight waves 512 (256), and goes through W.per blocks of 32
// of the columns that see them: their q as two fp16 parts from LDS (the attention's own products, aeth_attn_kv8_dev.hpp), the exponentials
// summed in registers over the blocks and at the end over the lanes. 32 / 8 heads of 128, a 2000-token prompt: 55 µs, 0.30 PFLOP/s of the formula
// (QKᵀ once), 0.60 of the matrix units'. A block takes 4170 cycles, its products 2050 of them on each matrix unit and 3370 of instructions
// beside them: an exponential and three more for each of 64 keys and 32 columns a lane pair, and making q's parts. The clock falls to 1.9 GHz.
// The first block comes some 6500 cycles late (the keys; 2500 more with loads of 8 bytes a lane).
template <int HD>
__global__ void __launch_bounds__(512, 2) k_kv8_weigh(A8 A, Weigh W) {
    constexpr int GK = sv_group(HD), NT = GK / 256, KS = HD / 16, KF = 1040, E = HD / 16, EV = E < 8 ? E : 8;
    __shared__ __attribute__((aligned(16))) char qb[2][2 * KS * KF];
    __shared__ __attribute__((aligned(16))) float4 col[2][32];  // scale of a product, maximum, 1 / sum, the key behind the last one it sees
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Workgroups go to the eight dies in turn: a KV head stays on one where there are eight. There are none without work, which
    // are not spread evenly and leave two on some CUs (with a third of them: 2000 tokens of 32 / 8 heads 106 µs).
    const int h = blockIdx.x % A.nkv, len = A.max_len, past = len - A.n;
    int group = W.first, chunk = blockIdx.x / A.nkv;
    if (chunk < W.full * W.chunks) {
        group += chunk / W.chunks;
        chunk %= W.chunks;
    } else {
        group += W.full;
        chunk -= W.full * W.chunks;
        for (int count; chunk >= (count = sv_count(A, W, group, GK)); chunk -= count) group++;
    }
    const int k0 = GK * group + 32 * NT * w;  // the wave's first key
    const Seen sees = sv_seen(A.n, A.G, len, A.window, GK * (int64_t)group, GK);
    const int b0 = chunk * W.per, b1 = min(b0 + W.per, sees.blocks);

    float acc[NT][16];
#pragma unroll
    for (int T = 0; T < NT; T++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[T][i] = 0.0f;

    if (b0 < b1) {  // (uniform)
        // a block of columns: 16 threads take one, E dimensions each
        const int sc = tid >> 4, sj = tid & 15;
        float y[E];
        float2 mi;
        int hi;             // the key behind the last one it sees
        // the column to fetch: its query and head, its q and statistics
        int x = sees.x_beg + 32 * b0 + sc, qi = x / A.G, qg = x % A.G;
        const int step_i = 32 / A.G, step_g = 32 % A.G;
        const float* src = A.q + (int64_t)qi * A.q_stride + (int64_t)(h * A.G + qg) * HD + E * sj;
        const int64_t step_src = step_i * A.q_stride + step_g * HD, wrap_src = A.q_stride - (int64_t)A.G * HD;
        const float2* stat = (const float2*)A.stat + (int64_t)h * A.cols;
        auto fetch = [&]() {
            const bool real = x < sees.x_end;  // past the end: some column, masked
            const float* p = real ? src : A.q + (int64_t)h * A.G * HD + E * sj;
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4 v;
                if (A.qvec) v = *(const float4*)(p + e);
                else v = make_float4(p[e], p[e + 1], p[e + 2], p[e + 3]);
                y[e] = v.x;
                y[e + 1] = v.y;
                y[e + 2] = v.z;
                y[e + 3] = v.w;
            }
            mi = stat[real ? x : 0];
            hi = real ? past + qi + 1 : 0;
            x += 32;
            qi += step_i;
            qg += step_g;
            src += step_src;
            if (qg >= A.G) {
                qg -= A.G;
                qi++;
                src += wrap_src;
            }
        };
        auto stage = [&](int buf) {
            uint32_t mb = 0;
#pragma unroll
            for (int e = 0; e < E; e++) mb = max(mb, __float_as_uint(y[e]) & 0x7FFFFFFFu);
            mb = kv8_umax<16>(mb);
            const int e2 = a8_exponent(__uint_as_float(mb)) - 8;  // the largest below 2^15
            // a row that is NaN (its sum is; an infinity or NaN in q makes it so): products that are NaN, so that a masked key's can be left out
            const bool nan = mi.y != mi.y;
            const float f = nan ? mi.y : a8_pow2(e2);
#pragma unroll
            for (int e = 0; e < E; e += EV) {
                typedef _Float16 part __attribute__((ext_vector_type(EV)));
                part hi, lo;
#pragma unroll
                for (int i = 0; i < EV; i++) {
                    const float v = y[e + i] * f;
                    hi[i] = (_Float16)v;
                    lo[i] = (_Float16)(v - (float)hi[i]);
                }
                const int dim = E * sj + e;
                char* dst = qb[buf] + (2 * (dim >> 5) + (dim >> 3 & 1)) * KF + (sc + 32 * (dim >> 4 & 1)) * 16 + 2 * (dim & 7);  // as the keys' order
                *(part*)dst = hi;
                *(part*)(dst + KS * KF) = lo;
            }
            if (sj == 0) {
                const float qs = a8_pow2(-e2) * (1.4426950408889634f / sqrtf((float)HD));
                col[buf][sc] = make_float4(nan ? 1.0f : qs, nan ? 0.0f : mi.x, nan ? 1.0f : mi.y, __int_as_float(hi));
            }
        };
        fetch();
        // keys: lane (key l%32, half l/32) of fragments (T, 2·s) and (T, 2·s + 1) holds eight each of the dimensions 32·s + 16·half .. + 15
        const uint8_t* p = A.cache + ((int64_t)h * A.tiles + min(k0, len - 1) / KV8_TILE) * aeth_kv8_tile_bytes(HD);
        a8_h8 kf[NT][KS];
        float sk[NT];
#pragma unroll
        for (int T = 0; T < NT; T++) {
            const int half = NT == 2 ? 32 * T : k0 & 32;  // of a tile
            const int st = half + 8 * ((lane >> 2) & 3) + 4 * hf + (lane & 3);
            const float ks = *(const float*)(p + 2 * KV8_TILE * HD + 4 * st), vs = *(const float*)(p + 2 * KV8_TILE * HD + 4 * (KV8_TILE + st));
            sk[T] = fabsf(vs) < INFINITY ? ks : __uint_as_float(0x7FC00000u);
#pragma unroll
            for (int s = 0; s < KS / 2; s++) {
                const uint4 k = *(const uint4*)(p + (half + c) * HD + 32 * s + 16 * hf);
                const a8_h4 a = a8_half4(k.x), b = a8_half4(k.y), d = a8_half4(k.z), e = a8_half4(k.w);
                kf[T][2 * s] = (a8_h8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
                kf[T][2 * s + 1] = (a8_h8){d[0], d[1], d[2], d[3], e[0], e[1], e[2], e[3]};
            }
        }
        // Some column of the blocks [w0, w1) sees a key of the wave. (At a prompt's diagonal half of the waves see none, and the others have
        // the SIMD to themselves.)
        const int64_t d0 = (int64_t)(k0 - past) * A.G - sees.x_beg, d1 = (int64_t)(k0 - past + 32 * NT - 1 + A.window) * A.G - sees.x_beg;
        const int w0 = (int)min(max(d0 >> 5, (int64_t)b0), (int64_t)b1);
        const int w1 = A.window > 0 ? (int)min(max((d1 + 31) >> 5, (int64_t)w0), (int64_t)b1) : b1;
        // the first and last query of a block: every column of it sees the keys [all_lo, all_hi)
        int x0 = sees.x_beg + 32 * w0, i_first = x0 / A.G, g_first = x0 % A.G;
        a8_f16 s[NT];       // a block's scores, from one block to the next
#pragma unroll
        for (int T = 0; T < NT; T++) s[T] = (a8_f16){};
        float4 cl = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto weigh = [&](float& a, float s, const float4& of) { a = fmaf(__builtin_amdgcn_exp2f(fmaf(s, of.x, -of.y)), of.z, a); };
        // The next block's columns are staged, and those behind them fetched, by the first four waves before their products and by
        // the others, one on each SIMD with them, behind: of two waves one has products for the matrix unit
        auto ahead = [&](int b, int buf) {
            if (b + 1 >= b1) return;  // (uniform)
            stage(buf ^ 1);
            if (b + 2 < b1) fetch();
        };
        stage(0);
        if (b0 + 1 < b1) fetch();
        __syncthreads();
        int b = b0;
        auto pass = [&](int end) {
            for (; b < end; b++) {
                ahead(b, (b - b0) & 1);
                __syncthreads();
            }
        };
        pass(w0);
        for (; b < w1; b++) {
            const int buf = (b - b0) & 1;
            if (w < 4) ahead(b, buf);
            const char* qp = qb[buf] + lane * 16;
            const float4 of = cl;
            cl = col[buf][c];
            // The products of a block, and between them one by one the exponentials of the block before (before the first: of nothing,
            // times 0): they run on different units, a product waits for the one before the last, and a wave issues in order
            a8_f16 d[NT];
            a8_h8 ql[2] = {*(const a8_h8*)(qp + KS * KF), *(const a8_h8*)(qp + (KS + 1) * KF)}, qh[2] = {*(const a8_h8*)qp, *(const a8_h8*)(qp + KF)};
            a8_unroll<2 * KS * NT>([&](auto mm) {
                constexpr int m = mm, T = m % NT, low = m / NT % 2 == 0, ks = m / (2 * NT);
                constexpr int first = 8 * m / KS, count = 8 * (m + 1) / KS - first;
                __builtin_amdgcn_sched_barrier(0);
                a8_h8& q = low ? ql[ks & 1] : qh[ks & 1];
                d[T] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[T][ks], q, low && ks == 0 ? (a8_f16){} : d[T], 0, 0, 0);
                if constexpr (T == NT - 1 && ks + 2 < KS) q = *(const a8_h8*)(qp + ((low ? KS : 0) + ks + 2) * KF);
                a8_unroll<count>([&](auto e) {
                    constexpr int i = first + e;
                    weigh(acc[i / 16][i % 16], s[i / 16][i % 16], of);
                    asm volatile("" : "+v"(acc[i / 16][i % 16]));  // here, and not behind the next branch, where it is used
                });
            });
            const int x1 = min(x0 + 31, sees.x_end - 1), i_last = i_first + (g_first + x1 - x0) / A.G;
            const int all_hi = x0 + 32 > sees.x_end ? 0 : past + i_first + 1, all_lo = A.window > 0 ? past + i_last + 1 - A.window : 0;
#pragma unroll
            for (int T = 0; T < NT; T++)
                a8_unroll<16>([&](auto at) {
                    constexpr int i = at;
                    s[T][i] = d[T][i] * a8_row<i>(sk[T]);
                });
            if (k0 + 32 * NT > all_hi) {  // (uniform) some key is behind a column's last
                const int hi = __float_as_int(cl.w) - k0 - 4 * hf;
#pragma unroll
                for (int T = 0; T < NT; T++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[T][i] = 32 * T + 8 * (i >> 2) + (i & 3) < hi ? s[T][i] : -INFINITY;
            }
            if (k0 < all_lo) {  // (uniform) some key is before a window
                const int lo = max(__float_as_int(cl.w) - k0 - 4 * hf, -64) - A.window;  // (a column that sees no key here is masked above)
#pragma unroll
                for (int T = 0; T < NT; T++)
#pragma unroll
                    for (int i = 0; i < 16; i++) s[T][i] = 32 * T + 8 * (i >> 2) + (i & 3) >= lo ? s[T][i] : -INFINITY;
            }
            if (w >= 4) ahead(b, buf);
            __syncthreads();  // the next block's columns are there, this one's readers done
            x0 += 32;
            i_first += step_i;
            g_first += step_g;
            if (g_first >= A.G) {
                g_first -= A.G;
                i_first++;
            }
        }
#pragma unroll
        for (int T = 0; T < NT; T++)
#pragma unroll
            for (int i = 0; i < 16; i++) weigh(acc[T][i], s[T][i], cl);
        pass(b1);
    }
    // over the columns: the sum in every lane of a half, lane c keeps the one of register c
    float v = 0.0f;
#pragma unroll
    for (int T = 0; T < NT; T++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float a = acc[T][i];
            a += aeth_dpp_xor1f(a);
            a += aeth_dpp_xor2f(a);
            a += aeth_dpp_mirror8f(a);
            a += aeth_dpp_mirror16f(a);
            const auto z = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false, false);
            a = __uint_as_float(z[0]) + __uint_as_float(z[1]);
            v = c == 16 * T + i ? a : v;
        }
    if (c >= 16 * NT) return;
    const int key = k0 + 32 * (c >> 4) + 8 * (c >> 2 & 3) + 4 * hf + (c & 3);
    if (W.chunks > 1) {
        W.part[((int64_t)chunk * A.nkv + h) * W.keys + key - GK * (int64_t)W.first] = v;
        return;
    }
    const int64_t at = h * W.max_seq + key;
    if (key < len) W.weights[at] = W.prior ? W.prior[at] + v : v;
}

// weights = prior + the chunks' sums; groups of gk keys (2000 keys of 8 heads in up to 12 chunks 5.2 µs)
__global__ void __launch_bounds__(256) k_kv8_weigh_sum(A8 A, Weigh W, int gk) {
    const int t0 = blockIdx.x * 256, t = t0 + threadIdx.x, h = blockIdx.y, group = t0 / gk;
    int chunks = 0;
    if (A.n > 0 && group >= W.first) chunks = sv_count(A, W, group, gk);  // (uniform)
    if (t >= A.max_len) return;
    const int64_t at = h * W.max_seq + t;
    const float* part = W.part + h * W.keys + t - gk * (int64_t)W.first;
    float v = 0.0f;
#pragma unroll 4
    for (int z = 0; z < chunks; z++) v += part[(int64_t)z * A.nkv * W.keys];
    W.weights[at] = W.prior ? W.prior[at] + v : v;
}

// Columns whose scores are kept; more are formed again. 32 / 8 heads of 128, 20000 tokens, µs with kept / formed scores: 28 columns (7 queries)
// 32.3 / 38.8, 40 41.0 / 45.2, 48 44.2 / 44.7, 56 49.9 / 46.8, 64 54.0 / 47.1; 2000 tokens: 48 22.3 / 23.5, 64 26.7 / 23.5. A batch, of one query
// a sequence, keeps them however many query heads a KV head has.
constexpr int64_t SCORES = 48;
bool sv_scores(int64_t cols, bool batch) { return batch || cols <= SCORES; }

// sums of at most this many groups of keys, in `units` groups of all heads
int64_t sv_sums(int64_t units) { return 4 * (int64_t)aeth_num_cus() + units; }

// Blocks of columns a workgroup takes. A workgroup fills a CU (eight waves of more than 128 registers) and costs about two
// blocks beside its own (its keys, the sum over lanes), so: the least rounds·(per + 2) of one to four rounds of workgroups.
void sv_chunks(Weigh& W, int64_t n, int64_t G, int64_t nkv, int64_t hd, int64_t len, int64_t window) {
    const int64_t gk = sv_group((int)hd), cus = aeth_num_cus(), end = aeth_cdiv(len, gk), begin = window > 0 ? std::max<int64_t>(0, len - n + 1 - window) / gk : 0;
    auto blocks = [&](int64_t g) { return std::max<int64_t>(1, sv_seen((int)n, (int)G, (int)len, (int)window, gk * g, (int)gk).blocks); };
    // the groups before `some` are seen by every query; the others, as many as the queries and a window reach, are counted one by one
    const int64_t some = window > 0 ? begin : std::min<int64_t>(end, (len - n) / gk + 1);
    int64_t most = some > begin ? blocks(begin) : 1, all = (some - begin) * most;
    for (int64_t g = some; g < end; g++) {
        all += blocks(g);
        most = std::max(most, blocks(g));
    }
    const int64_t units = (end - begin) * nkv, fewest = aeth_cdiv(most, sv_sums(units) / units);
    int64_t best = most, least = INT64_MAX;
    for (int64_t rounds = 1; rounds <= 4; rounds++)
        for (int64_t more = 0; more < 3; more++) {
            const int64_t per = std::min(std::max(fewest, aeth_cdiv(all * nkv, rounds * cus) + more), most);
            int64_t wgs = (some - begin) * aeth_cdiv(most, per);
            for (int64_t g = some; g < end; g++) wgs += aeth_cdiv(blocks(g), per);
            const int64_t cost = aeth_cdiv(wgs * nkv, cus) * (per + 2);
            if (cost < least) {
                least = cost;
                best = per;
            }
        }
    W.per = (int)best;
    W.chunks = (int)aeth_cdiv(most, best);
    W.first = W.chunks > 1 ? (int)begin : 0;  // one chunk: every group, those that nothing sees for their prior
    W.keys = (end - W.first) * gk;
    W.full = (int)(W.chunks == 1 ? end : some - begin);  // (begin > 0 with a window only)
    W.wgs = W.full * W.chunks;
    for (int64_t g = W.first + W.full; g < end; g++) W.wgs += (int)aeth_cdiv(blocks(g), best);
}

// the workspace's parts, bytes from its start: the attention's own, columns' statistics, scores or sums by chunk
struct WeighWs {
    int64_t stat, rest, end;
};
WeighWs sv_weigh_ws(int64_t seqs, int64_t n, int64_t nq, int64_t nkv, int64_t hd, int64_t len) {
    const int64_t G = nq / nkv, cols = n * G;
    WeighWs w;
    w.stat = aeth_attn_kv8_ws(seqs, n, nq, nkv, hd, len);
    w.rest = w.stat + aeth_cdiv(seqs * nkv * cols * 8, 16) * 16;
    // a smaller call may keep scores where the largest does not
    const int64_t scores = seqs * nkv * std::min(cols, std::max(G, SCORES)) * aeth_cdiv(len, KV8_TILE) * KV8_TILE;
    const int64_t gk = sv_group((int)hd), sums = cols > SCORES ? sv_sums(nkv * aeth_cdiv(len, gk)) * gk : 0;
    w.end = w.rest + std::max(scores, sums) * 4;
    return w;
}

template <int HD, int KT>
void sv_weigh_kept(const A8& A, const Weigh& W, int64_t seqs, hipStream_t s) {
    const dim3 block(256);
    const int64_t pieces = A.nkv * aeth_cdiv(A.max_len, 256 * KT), cols = (int64_t)A.nkv * A.cols, joins = aeth_cdiv(cols * (HD / 4), 256);
    auto grid = [&](int64_t n) { return dim3((unsigned)n, (unsigned)seqs); };
    if (A.chunks == 1) hipLaunchKernelGGL((k_kv8_weigh_scores<HD, KT>), grid(pieces), block, 0, s, A, W);
    else if (a8_merge_is_some(A, seqs)) hipLaunchKernelGGL((k_kv8_join_weigh<HD, true, KT>), grid(joins + pieces), block, 0, s, A, W, (int)joins);
    else hipLaunchKernelGGL((k_kv8_join_weigh<HD, false, KT>), grid(cols + pieces), block, 0, s, A, W, (int)cols);
}

template <int HD>
int sv_weigh(A8 A, Weigh W, const Form& f, int64_t seqs, bool scores, hipStream_t s) {
    if (scores) {
        hipLaunchKernelGGL((k_attn8<HD, A8_STAT | A8_SCORE>), dim3((unsigned)(A.nkv * A.ncb), (unsigned)seqs, (unsigned)A.chunks), dim3(256), 0, s, A);
        AETH_LAUNCH_CHECK();
        // four keys a thread where one each makes more workgroups than the CUs hold at once
        if (A.nkv * aeth_cdiv(A.max_len, 256) * seqs > 8 * (int64_t)aeth_num_cus()) sv_weigh_kept<HD, 4>(A, W, seqs, s);
        else sv_weigh_kept<HD, 1>(A, W, seqs, s);
        AETH_LAUNCH_CHECK();
        return AETH_OK;
    }
    const int rc = a8_launch<HD, A8_STAT>(A, f, seqs, s);
    if (rc) return rc;
    hipLaunchKernelGGL(k_kv8_weigh<HD>, dim3((unsigned)(A.nkv * W.wgs)), dim3(512), 0, s, A, W);
    AETH_LAUNCH_CHECK();
    if (W.chunks > 1) {
        hipLaunchKernelGGL(k_kv8_weigh_sum, dim3((unsigned)aeth_cdiv(A.max_len, 256), (unsigned)A.nkv), dim3(256), 0, s, A, W, sv_group(HD));
        AETH_LAUNCH_CHECK();
    }
    return AETH_OK;
}

int sv_attn_weights(const char* what, const float* q, int64_t q_stride, const void* cache, int64_t stride, const int* lens, int64_t seqs, int64_t n,
                    int64_t nq, int64_t nkv, int64_t hd, int64_t max_seq, int64_t max_len, int64_t window, float* out, const float* prior, float* weights,
                    void* ws, int64_t ws_bytes, hipStream_t s) {
    if (!weights || (((uintptr_t)weights | (uintptr_t)prior) & 3)) return aeth_set_error(AETH_EINVAL, "%s: bad argument (weights)", what);
    if (n == 0) q = out = weights;  // no query, no row: either may be NULL
    int rc = aeth_attn_kv8_check(what, q, q_stride, cache, seqs, n, nq, nkv, hd, max_seq, max_len, window, out, ws);
    if (rc) return rc;
    if (nkv * aeth_cdiv(max_len, 256) + nq * n > (int64_t)1 << 23)  // workgroups of up to 512 threads within the grid's 2^32
        return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld positions of %lld heads in one call", what, (long long)max_len, (long long)nkv);
    const WeighWs at = sv_weigh_ws(seqs, n, nq, nkv, hd, max_len);
    rc = aeth_attn_kv8_check_ws(what, ws, ws_bytes, at.end);
    if (!rc && lens) rc = aeth_attn_kv8_check_slices(what, seqs, stride, nkv, hd, max_seq);
    if (rc) return rc;
    const int64_t bytes = seqs * nkv * max_seq * 4;  // below 2^16·2^12·2^30·2^2
    if (prior && prior != weights && (uintptr_t)prior < (uintptr_t)weights + (uint64_t)bytes && (uintptr_t)weights < (uintptr_t)prior + (uint64_t)bytes)
        return aeth_set_error(AETH_EINVAL, "%s: the weights before and after overlap", what);
    if (seqs == 0 || max_len == 0) return AETH_OK;
    Weigh W = {};
    W.prior = prior;
    W.weights = weights;
    W.max_seq = max_seq;
    W.part = (float*)((char*)ws + at.rest);
    A8 A = a8_args(q, q_stride, cache, stride, lens, 0, n, nq, nkv, max_seq, max_len, window, out, ws);
    if (n == 0) {  // no query: the weights as they were
        hipLaunchKernelGGL(k_kv8_weigh_sum, dim3((unsigned)aeth_cdiv(max_len, 256), (unsigned)nkv), dim3(256), 0, s, A, W, 256);
        AETH_LAUNCH_CHECK();
        return AETH_OK;
    }
    const Form f = a8_form(seqs, n, A.G, nkv, hd, max_len, A.window, lens != nullptr);
    a8_take(A, f);
    A.stat = (float*)((char*)ws + at.stat);
    const bool scores = sv_scores(A.cols, lens != nullptr);
    A.scores = W.part;
    A.score_tiles = (int)aeth_cdiv(max_len, KV8_TILE);
    if (!scores) sv_chunks(W, n, A.G, nkv, hd, max_len, A.window);
    if (hd == 64) return sv_weigh<64>(A, W, f, seqs, scores, s);
    if (hd == 128) return sv_weigh<128>(A, W, f, seqs, scores, s);
    return sv_weigh<256>(A, W, f, seqs, scores, s);
}

}  // namespace

extern "C" AETH_API int64_t aeth_attn_kv8_shared_ws_bytes(int64_t n_seqs, int64_t n_heads, int64_t kv_heads, int64_t head_dim, int64_t prefix_len,
                                                          int64_t max_len) {
    if (aeth_attn_kv8_ws_bytes(n_seqs, 1, n_heads, kv_heads, head_dim, max_len) < 0 || prefix_len < 0 || prefix_len > KV8_MAX_SEQ) {
        aeth_set_error(AETH_EINVAL, "aeth_attn_kv8_shared_ws_bytes: bad shape");
        return -1;
    }
    return sv_own_ws(n_seqs, n_heads, kv_heads, head_dim) + (prefix_len > 0 ? sv_prefix_ws(n_seqs, n_heads, kv_heads, head_dim) : 0);
}

extern "C" AETH_API int aeth_attn_kv8_shared(const float* d_q, int64_t q_stride, const void* d_prefix, int64_t prefix_seq, int64_t prefix_len,
                                             const void* d_layers, int64_t layer_stride, const int32_t* d_lens, int64_t n_seqs, int64_t n_heads,
                                             int64_t kv_heads, int64_t head_dim, int64_t max_seq, int64_t max_len, int64_t window, float* d_out,
                                             void* d_ws, int64_t ws_bytes, void* stream) {
    const char* what = "aeth_attn_kv8_shared";
    if (!d_lens || ((uintptr_t)d_lens & 3) || max_len < 1) return aeth_set_error(AETH_EINVAL, "%s: bad argument (lengths)", what);
    if (prefix_len < 0 || prefix_len > prefix_seq || prefix_seq > KV8_MAX_SEQ || (prefix_len > 0 && (!d_prefix || ((uintptr_t)d_prefix & 15))))
        return aeth_set_error(AETH_EINVAL, "%s: bad argument (a prefix of %lld tokens in a slice of %lld, 16-byte aligned)", what, (long long)prefix_len,
                              (long long)prefix_seq);
    int rc = aeth_attn_kv8_check(what, d_q, q_stride, d_layers, n_seqs, 1, n_heads, kv_heads, head_dim, max_seq, max_len, window, d_out, d_ws);
    if (!rc) rc = aeth_attn_kv8_check_slices(what, n_seqs, layer_stride, kv_heads, head_dim, max_seq);
    if (!rc && prefix_len > KV8_MAX_SEQ - max_len)
        rc = aeth_set_error(AETH_EINVAL, "%s: %lld tokens behind %lld", what, (long long)max_len, (long long)prefix_len);
    if (!rc && n_seqs * kv_heads * aeth_cdiv(n_heads / kv_heads, 16) > (int64_t)1 << 22)  // workgroups of 256 threads within the grid's 2^32
        rc = aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld sequences of %lld heads in one call", what, (long long)n_seqs, (long long)n_heads);
    if (rc || n_seqs == 0) return rc;
    const int64_t own = sv_own_ws(n_seqs, n_heads, kv_heads, head_dim);
    rc = aeth_attn_kv8_check_ws(what, d_ws, ws_bytes, own + (prefix_len > 0 ? sv_prefix_ws(n_seqs, n_heads, kv_heads, head_dim) : 0));
    if (rc) return rc;
    const int64_t reach = window < prefix_len + max_len ? window : 0;  // one that reaches past the first key masks nothing
    A8 P = a8_args(d_q, q_stride, d_prefix, 0, nullptr, 0, n_seqs, n_heads, kv_heads, prefix_seq, prefix_len, 0, nullptr, (char*)d_ws + own);
    P.window = (int)reach;
    P.own_lens = d_lens;
    P.own_max = (int)max_len;
    const A8 O = a8_args(d_q, q_stride, d_layers, layer_stride, d_lens, 0, 1, n_heads, kv_heads, max_seq, max_len, reach, d_out, d_ws);
    if (head_dim == 64) return sv_shared<64>(P, O, n_seqs, (hipStream_t)stream);
    if (head_dim == 128) return sv_shared<128>(P, O, n_seqs, (hipStream_t)stream);
    return sv_shared<256>(P, O, n_seqs, (hipStream_t)stream);
}

extern "C" AETH_API int64_t aeth_attn_kv8_weights_ws_bytes(int64_t n_seqs, int64_t n, int64_t n_heads, int64_t kv_heads, int64_t head_dim,
                                                           int64_t max_len) {
    if (aeth_attn_kv8_ws_bytes(n_seqs, n, n_heads, kv_heads, head_dim, max_len) < 0) {
        aeth_set_error(AETH_EINVAL, "aeth_attn_kv8_weights_ws_bytes: bad shape");
        return -1;
    }
    int64_t all;  // the scores of the largest, as sv_weigh_ws has them
    if (!aeth_mul_ok(n_seqs * kv_heads, std::min(n * (n_heads / kv_heads), std::max(n_heads / kv_heads, SCORES)), &all) ||
        !aeth_mul_ok(all, max_len + KV8_TILE, &all) || all > (int64_t)1 << 58) {
        aeth_set_error(AETH_EINVAL, "aeth_attn_kv8_weights_ws_bytes: bad shape");
        return -1;
    }
    return sv_weigh_ws(n_seqs, n, n_heads, kv_heads, head_dim, max_len).end;
}

extern "C" AETH_API int aeth_attn_kv8_weights(const float* d_q, int64_t q_stride, const void* d_layer, int64_t n, int64_t n_heads, int64_t kv_heads,
                                              int64_t head_dim, int64_t max_seq, int64_t seq, int64_t window, float* d_out, const float* d_prior,
                                              float* d_weights, void* d_ws, int64_t ws_bytes, void* stream) {
    return sv_attn_weights("aeth_attn_kv8_weights", d_q, q_stride, d_layer, 0, nullptr, 1, n, n_heads, kv_heads, head_dim, max_seq, seq, window, d_out,
                           d_prior, d_weights, d_ws, ws_bytes, (hipStream_t)stream);
}

extern "C" AETH_API int aeth_attn_kv8_weights_batch(const float* d_q, int64_t q_stride, const void* d_layers, int64_t layer_stride, const int32_t* d_lens,
                                                    int64_t n_seqs, int64_t n_heads, int64_t kv_heads, int64_t head_dim, int64_t max_seq,
                                                    int64_t max_len, int64_t window, float* d_out, const float* d_prior, float* d_weights, void* d_ws,
                                                    int64_t ws_bytes, void* stream) {
    const char* what = "aeth_attn_kv8_weights_batch";
    if (!d_lens || ((uintptr_t)d_lens & 3) || max_len < 1) return aeth_set_error(AETH_EINVAL, "%s: bad argument (lengths)", what);
    return sv_attn_weights(what, d_q, q_stride, d_layers, layer_stride, d_lens, n_seqs, 1, n_heads, kv_heads, head_dim, max_seq, max_len, window, d_out,
                           d_prior, d_weights, d_ws, ws_bytes, (hipStream_t)stream);
}
