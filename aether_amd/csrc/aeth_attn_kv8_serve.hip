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
// known behind the attention. Up to 64 columns its workgroups also leave their scores, 4 bytes a column and key where a
// key's codes are 2·hd + 8 (k_kv8_weigh_scores); of more the scores are formed once more from the keys (k_kv8_weigh), where they are summed
// over columns in registers: no score reaches memory. Every sum has a fixed order.
#include "aeth_attn_kv8_dev.hpp"

namespace {

// ── a shared prefix ───────────────────────────────────────────────────────

// Joins a column's parts of the prefix (P, blocks of cw columns) and of its own tokens (O, of 16): HD/4 lanes of four dimensions, GR of such
// groups take every GR-th part.
template <int HD, int GR>
__global__ void __launch_bounds__(256) k_attn8_join(A8 P, int cw, A8 O) {
    constexpr int L = HD / 4, CW = 256 / (L * GR);  // columns a workgroup
    __shared__ __attribute__((aligned(16))) float sum[GR > 1 ? GR : 1][GR > 1 ? HD : 4];
    const int tid = threadIdx.x, d = 4 * (tid % L), grp = tid / L % GR, seq = blockIdx.y;
    const int unit = blockIdx.x * CW + tid / (L * GR);
    if (unit >= O.nkv * O.G) return;  // (uniform where GR > 1)
    const int h = unit / O.G, g = unit % O.G;
    int beg, end;
    a8_tiles(O, a8_len(O, seq), g / 16 * 16, 16, beg, end);
    const int live_o = max(1, (end - beg + O.tpc - 1) / O.tpc);
    a8_tiles<A8_FLAT>(P, 0, 0, 0, beg, end);
    const int live_p = (end - beg + P.tpc - 1) / P.tpc, live = live_p + live_o;
    const int x = seq * O.G + g;
    const int64_t step_p = (int64_t)cw * (HD + 2), step_o = 16 * (HD + 2);
    const float* part_p = P.ws + (int64_t)(h * P.ncb + x / cw) * P.chunks * step_p;
    const float* part_o = O.ws + (int64_t)((seq * O.nkv + h) * O.ncb + g / 16) * O.chunks * step_o;
    const int cp = x % cw, co = g % 16;
    auto stat = [&](int k) { return *(const float2*)(k < live_p ? part_p + k * step_p + cw * HD + 2 * cp : part_o + (k - live_p) * step_o + 16 * HD + 2 * co); };
    auto value = [&](int k) { return *(const a8_f4*)(k < live_p ? part_p + k * step_p + cp * HD + d : part_o + (k - live_p) * step_o + co * HD + d); };
    float M = -INFINITY, S = 0.0f;
    if constexpr (GR > 1) {
        const int lane = tid & 63;
        for (int k = lane; k < live; k += 64) M = fmaxf(M, stat(k).x);
        M = aeth_wave_max(M);
        for (int k = lane; k < live; k += 64) {
            const float2 ml = stat(k);
            S += (ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M)) * ml.y;
        }
        S = aeth_wave_sum(S);
    } else {
#pragma unroll 4
        for (int k = 0; k < live; k++) M = fmaxf(M, stat(k).x);
    }
    a8_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int k = grp; k < live; k += GR) {
        const float2 ml = stat(k);
        const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
        acc += value(k) * w;
        if (GR == 1) S += w * ml.y;
    }
    float* dst = O.out + (int64_t)seq * ((int64_t)O.nq * HD) + (int64_t)unit * HD;
    if constexpr (GR > 1) {
        *(a8_f4*)&sum[grp][d] = acc;
        __syncthreads();
        if (tid >= HD) return;
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < GR; i++) y += sum[i][tid];
        dst[tid] = S == 0.0f ? 0.0f : y * (1.0f / S);
    } else {
        acc = S == 0.0f ? (a8_f4){0.0f, 0.0f, 0.0f, 0.0f} : acc * (1.0f / S);
        if (O.ovec) *(a8_f4*)(dst + d) = acc;
        else dst[d] = acc[0], dst[d + 1] = acc[1], dst[d + 2] = acc[2], dst[d + 3] = acc[3];
    }
}

// The prefix's form: a8_form's reckoning for columns that all see `span` tiles
Form sv_prefix_form(int64_t cols, int64_t nkv, int64_t hd, int64_t span) {
    const int64_t cus = aeth_num_cus();
    const Form small = a8_split(16, nkv * aeth_cdiv(cols, 16), span, 2 * cus, 4);
    if (hd > 128 || cols <= 64) return small;
    const double c = (double)cus;
    Form best = small;
    double least = INFINITY;
    for (int64_t cw = 16; cw <= (hd == 128 ? 256 : 128); cw = std::max<int64_t>(128, 2 * cw)) {
        const int64_t units = nkv * aeth_cdiv(cols, cw);
        const double tiles = (double)units * (double)span;
        for (int64_t target : {(int64_t)0, cus, 2 * cus, 4 * cus}) {
            if (target > (cw == 16 ? 4 : cw == 128 ? 2 : 1) * cus) continue;
            const Form f = a8_split(cw, units, span, std::max<int64_t>(1, target), cw == 16 ? 4 : 8);
            const int64_t wgs = units * f.chunks;
            const double w = tiles / c, tpc = (double)std::min<int64_t>(f.tpc, span);
            const double u = (double)aeth_cdiv(wgs, cus), q = u * (tiles / (double)wgs);
            const double own = std::max(tpc, w);
            double t = cw == 256   ? 12.0 + 2.8 * own + 1.5 * std::max(0.0, w - 0.4 * own)
                       : cw == 128 ? (hd == 128 ? std::max(8.0 + 2.3 * tpc, 22.0 + 1.96 * w) : std::max(7.0 + 1.53 * tpc, 15.0 + 1.25 * w))
                       : hd == 128 ? std::max(5.5 + 0.45 * tpc, 6.0 + 0.33 * q + 4.5 * std::ceil(u / 3.0))
                                   : std::max(5.0 + 0.3 * tpc, 5.0 + 0.185 * q + 2.8 * std::ceil(u / 4.0));
            t += (cw == 16 ? 2e-6 : 1e-6) * (double)(nkv * cols * f.chunks) * (double)(hd + 2);
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
    if (hd == 128 && cols > 64) most = std::max(most, need(256, cus));
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
        fp = sv_prefix_form(P.cols, P.nkv, HD, span);
    }
    a8_take(P, fp);
    if (P.chunks > 0) {
        const int rc = a8_launch<HD, A8_FLAT | A8_PART>(P, fp, 1, s);
        if (rc) return rc;
    }
    hipLaunchKernelGGL((k_attn8<HD, A8_PART>), dim3((unsigned)(O.nkv * O.ncb), (unsigned)seqs, (unsigned)O.chunks), dim3(256), 0, s, O);
    AETH_LAUNCH_CHECK();
    const int64_t cols = (int64_t)O.nkv * O.G;
    constexpr int GR = 1024 / HD;
    if (P.chunks + O.chunks <= 8) hipLaunchKernelGGL((k_attn8_join<HD, 1>), dim3((unsigned)aeth_cdiv(cols, GR), (unsigned)seqs), dim3(256), 0, s, P, fp.cw, O);
    else hipLaunchKernelGGL((k_attn8_join<HD, GR>), dim3((unsigned)cols, (unsigned)seqs), dim3(256), 0, s, P, fp.cw, O);
    AETH_LAUNCH_CHECK();
    return AETH_OK;
}

// ── the weights that tokens receive ───────────────────────────────────────

struct Weigh {
    const float* prior;  // [seqs][nkv][max_seq]; nullptr: zeros
    float* weights;
    int64_t max_seq;
    float* part;         // k_kv8_weigh in several chunks of columns: [chunks][nkv][keys]
    int chunks;
    int64_t keys;        // of a row of part: a multiple of 256
};

// From the scores of up to a few hundred columns: 1024 keys a workgroup
__global__ void __launch_bounds__(256) k_kv8_weigh_scores(A8 A, Weigh W) {
    constexpr int CB = 64;
    __shared__ float2 col[CB];  // maximum, 1 / sum
    const int tid = threadIdx.x, h = blockIdx.y, seq = blockIdx.z;
    const int len = a8_len(A, seq), t0 = blockIdx.x * 1024;
    if (t0 >= len) return;  // (uniform)
    const int64_t unit = (int64_t)seq * A.nkv + h, row = 64 * (int64_t)A.score_tiles;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < A.cols; c0 += CB) {
        const int count = min(CB, A.cols - c0);
        __syncthreads();
        if (tid < count) {
            const float2 ml = *(const float2*)(A.stat + 2 * (unit * A.cols + c0 + tid));
            col[tid] = make_float2(ml.x, 1.0f / ml.y);
        }
        __syncthreads();
        for (int c = 0; c < count; c++) {
            const int hi = len - A.n + (c0 + c) / A.G + 1, lo = A.window > 0 ? hi - A.window : 0;  // (uniform)
            const float* src = A.scores + (unit * A.cols + c0 + c) * row;
            const float2 mi = col[c];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int t = t0 + tid + 256 * j;
                if (t >= lo && t < hi) acc[j] = fmaf(__builtin_amdgcn_exp2f(src[t] - mi.x), mi.y, acc[j]);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int64_t t = t0 + tid + 256 * j, at = unit * W.max_seq + t;
        if (t < len) W.weights[at] = W.prior ? W.prior[at] + acc[j] : acc[j];
    }
}

// Many columns: a wave keeps 64 keys (one tile) as fp16 in registers, its workgroup 256, and goes through its columns 32 at a
// time: their q as two fp16 parts from LDS (aeth_attn_kv8_dev.hpp: the same products as the attention's), the scores' exponentials summed
// in registers over the blocks of columns and at the end over the lanes.
template <int HD>
__global__ void __launch_bounds__(256, 2) k_kv8_weigh(A8 A, Weigh W) {
    constexpr int KS = HD / 16, KF = 1040, E = HD / 8;
    __shared__ __attribute__((aligned(16))) char qb[2][2 * KS * KF];
    __shared__ __attribute__((aligned(16))) float4 col[2][32];  // scale of a product, maximum, 1 / sum, the key behind the last one it sees
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.y, chunk = blockIdx.z, len = A.max_len, k0 = 256 * blockIdx.x;
    const int last = (len - 1) >> 6, t = 4 * blockIdx.x + w, tl = min(t, last);
    // the columns that see a key of the workgroup, those of this chunk
    const int past = len - A.n;  // keys before the first query
    const int i0 = max(0, k0 - past), i1 = A.window > 0 ? (int)min((int64_t)A.n, (int64_t)min(k0 + 256, len) + A.window - 1 - past) : A.n;
    const int nb = i1 > i0 ? ((i1 - i0) * A.G + 31) / 32 : 0, per = (nb + W.chunks - 1) / W.chunks;
    const int b0 = chunk * per, b1 = min(b0 + per, nb);
    const int x_beg = i0 * A.G, x_end = i1 * A.G;

    float acc[2][16];
#pragma unroll
    for (int T = 0; T < 2; T++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[T][i] = 0.0f;

    if (b0 < b1) {  // (uniform)
        // keys: lane (key l%32, half l/32) of fragment (T, ks) holds eight dimensions
        const uint8_t* p = A.cache + ((int64_t)h * A.tiles + tl) * aeth_kv8_tile_bytes(HD);
        a8_h8 kf[2][KS];
        float sk[2];
#pragma unroll
        for (int T = 0; T < 2; T++) {
            const int st = 32 * T + 8 * ((lane >> 2) & 3) + 4 * hf + (lane & 3);
            const float ks = *(const float*)(p + 2 * KV8_TILE * HD + 4 * st), vs = *(const float*)(p + 2 * KV8_TILE * HD + 4 * (KV8_TILE + st));
            sk[T] = fabsf(vs) < INFINITY ? ks : __uint_as_float(0x7FC00000u);
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const uint2 k = *(const uint2*)(p + (32 * T + c) * HD + 16 * s + 8 * hf);
                const a8_h4 a = a8_half4(k.x), b = a8_half4(k.y);
                kf[T][s] = (a8_h8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
            }
        }
        // a block of columns: eight threads take one
        const int sc = tid >> 3, sj = tid & 7;
        float y[E];
        float2 ml;
        int qi = 0;
        bool real = false;
        auto fetch = [&](int b) {
            const int x = x_beg + 32 * b + sc, xc = min(x, x_end - 1);
            real = x < x_end;
            qi = xc / A.G;
            const float* src = A.q + (int64_t)qi * A.q_stride + (int64_t)(h * A.G + xc % A.G) * HD + E * sj;
#pragma unroll
            for (int e = 0; e < E; e += 4) {
                float4 v;
                if (A.qvec) v = *(const float4*)(src + e);
                else v = make_float4(src[e], src[e + 1], src[e + 2], src[e + 3]);
                y[e] = v.x;
                y[e + 1] = v.y;
                y[e + 2] = v.z;
                y[e + 3] = v.w;
            }
            ml = *(const float2*)(A.stat + 2 * ((int64_t)h * A.cols + xc));
        };
        auto stage = [&](int buf) {
            uint32_t mb = 0;
#pragma unroll
            for (int e = 0; e < E; e++) mb = max(mb, __float_as_uint(y[e]) & 0x7FFFFFFFu);
            mb = kv8_umax<8>(mb);
            const int e2 = a8_exponent(__uint_as_float(mb)) - 8;  // the largest below 2^15
            const float f = a8_pow2(e2);
#pragma unroll
            for (int e = 0; e < E; e += 8) {
                a8_h8 hi, lo;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float v = y[e + i] * f;
                    hi[i] = (_Float16)v;
                    lo[i] = (_Float16)(v - (float)hi[i]);
                }
                const int dim = E * sj + e;
                char* dst = qb[buf] + (dim >> 4) * KF + (sc + 32 * (dim >> 3 & 1)) * 16;
                *(a8_h8*)dst = hi;
                *(a8_h8*)(dst + KS * KF) = lo;
            }
            if (sj == 0) {
                // an infinity or NaN in q: every score NaN
                const float qs = mb >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : a8_pow2(-e2) * (1.4426950408889634f / sqrtf((float)HD));
                col[buf][sc] = make_float4(qs, ml.x, 1.0f / ml.y, __int_as_float(real ? past + qi + 1 : (int)0x80000000));
            }
        };
        fetch(b0);
        for (int b = b0; b < b1; b++) {
            const int buf = (b - b0) & 1;
            stage(buf);
            __syncthreads();  // (the other buffer's readers have passed the barrier before this one)
            if (b + 1 < b1) fetch(b + 1);
            const float4 cl = col[buf][c];
            a8_f16 s[2] = {(a8_f16){}, (a8_f16){}};
            const char* qp = qb[buf] + lane * 16;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const a8_h8 ql = *(const a8_h8*)(qp + (KS + ks) * KF), qh = *(const a8_h8*)(qp + ks * KF);
                s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[0][ks], ql, s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[1][ks], ql, s[1], 0, 0, 0);
                s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[0][ks], qh, s[0], 0, 0, 0);
                s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[1][ks], qh, s[1], 0, 0, 0);
            }
            // every column of the block sees the keys [all_lo, all_hi)
            const int x0 = x_beg + 32 * b, all_hi = x0 + 32 > x_end ? 0 : past + x0 / A.G + 1;
            const int all_lo = A.window > 0 ? past + min(x0 + 31, x_end - 1) / A.G + 1 - A.window : 0;
            const int hi = __float_as_int(cl.w), lo = A.window > 0 ? max(hi, 0) - A.window : 0;
            const bool masked = 64 * t < all_lo || 64 * t + 64 > all_hi;  // (uniform)
#pragma unroll
            for (int T = 0; T < 2; T++)
                a8_unroll<16>([&](auto at) {
                    constexpr int i = at;
                    float e = __builtin_amdgcn_exp2f(fmaf(s[T][i] * a8_row<i>(sk[T]), cl.x, -cl.y)) * cl.z;
                    if (masked) {
                        const int key = 64 * t + 32 * T + 8 * (i >> 2) + 4 * hf + (i & 3);
                        e = key >= lo && key < hi ? e : 0.0f;
                    }
                    acc[T][i] += e;
                });
        }
    }
    // over the columns: the sum in every lane of a half, lane c keeps the one of register c
    float v = 0.0f;
#pragma unroll
    for (int T = 0; T < 2; T++)
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
    const int key = 64 * t + 32 * (c >> 4) + 8 * (c >> 2 & 3) + 4 * hf + (c & 3);
    if (W.chunks > 1) {
        W.part[((int64_t)chunk * A.nkv + h) * W.keys + key] = v;
        return;
    }
    const int64_t at = h * W.max_seq + key;
    if (key < len) W.weights[at] = W.prior ? W.prior[at] + v : v;
}

// weights = prior + the chunks' sums
__global__ void __launch_bounds__(256) k_kv8_weigh_sum(Weigh W, int64_t len, int nkv) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int h = blockIdx.y;
    if (t >= len) return;
    const int64_t at = h * W.max_seq + t;
    float v = 0.0f;
    for (int z = 0; z < W.chunks; z++) v += W.part[((int64_t)z * nkv + h) * W.keys + t];
    W.weights[at] = W.prior ? W.prior[at] + v : v;
}

// columns whose scores are kept; more are formed again
constexpr int64_t SCORES = 64;
bool sv_scores(int64_t seqs, int64_t cols, bool batch) { return batch || cols <= SCORES; }

int64_t sv_chunks(int64_t cols, int64_t nkv, int64_t len) {
    const int64_t units = nkv * aeth_cdiv(len, 256);
    return std::max<int64_t>(1, std::min(aeth_cdiv(4 * (int64_t)aeth_num_cus(), units), aeth_cdiv(cols, 4 * 32)));
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
    const int64_t units = nkv * aeth_cdiv(len, 256), sums = cols > SCORES ? (4 * (int64_t)aeth_num_cus() + units) * 256 : 0;
    w.end = w.rest + std::max(scores, sums) * 4;
    return w;
}

template <int HD>
int sv_weigh(A8 A, Weigh W, const Form& f, int64_t seqs, bool scores, hipStream_t s) {
    const int rc = scores ? a8_launch<HD, A8_STAT | A8_SCORE>(A, f, seqs, s) : a8_launch<HD, A8_STAT>(A, f, seqs, s);
    if (rc) return rc;
    if (scores) {
        hipLaunchKernelGGL(k_kv8_weigh_scores, dim3((unsigned)aeth_cdiv(A.max_len, 1024), (unsigned)A.nkv, (unsigned)seqs), dim3(256), 0, s, A, W);
        AETH_LAUNCH_CHECK();
        return AETH_OK;
    }
    hipLaunchKernelGGL(k_kv8_weigh<HD>, dim3((unsigned)aeth_cdiv(A.max_len, 256), (unsigned)A.nkv, (unsigned)W.chunks), dim3(256), 0, s, A, W);
    AETH_LAUNCH_CHECK();
    if (W.chunks > 1) {
        hipLaunchKernelGGL(k_kv8_weigh_sum, dim3((unsigned)aeth_cdiv(A.max_len, 256), (unsigned)A.nkv), dim3(256), 0, s, W, (int64_t)A.max_len, A.nkv);
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
    if (nkv > 65535) return aeth_set_error(AETH_EUNSUPPORTED, "%s: %lld KV heads", what, (long long)nkv);
    const WeighWs at = sv_weigh_ws(seqs, n, nq, nkv, hd, max_len);
    rc = aeth_attn_kv8_check_ws(what, ws, ws_bytes, at.end);
    if (!rc && lens) rc = aeth_attn_kv8_check_slices(what, seqs, stride, nkv, hd, max_seq);
    if (rc) return rc;
    const int64_t bytes = seqs * nkv * max_seq * 4;  // below 2^16·2^12·2^30·2^2
    if (prior && prior != weights && (uintptr_t)prior < (uintptr_t)weights + (uint64_t)bytes && (uintptr_t)weights < (uintptr_t)prior + (uint64_t)bytes)
        return aeth_set_error(AETH_EINVAL, "%s: the weights before and after overlap", what);
    if (seqs == 0 || max_len == 0) return AETH_OK;
    Weigh W = {prior, weights, max_seq, (float*)((char*)ws + at.rest), 0, aeth_cdiv(max_len, 256) * 256};
    if (n == 0) {  // no query: the weights as they were
        hipLaunchKernelGGL(k_kv8_weigh_sum, dim3((unsigned)aeth_cdiv(max_len, 256), (unsigned)nkv), dim3(256), 0, s, W, max_len, (int)nkv);
        AETH_LAUNCH_CHECK();
        return AETH_OK;
    }
    A8 A = a8_args(q, q_stride, cache, stride, lens, 0, n, nq, nkv, max_seq, max_len, window, out, ws);
    const Form f = a8_form(seqs, n, A.G, nkv, hd, max_len, A.window, lens != nullptr);
    a8_take(A, f);
    A.stat = (float*)((char*)ws + at.stat);
    const bool scores = sv_scores(seqs, A.cols, lens != nullptr);
    A.scores = (float*)((char*)ws + at.rest);
    A.score_tiles = (int)aeth_cdiv(max_len, KV8_TILE);
    W.chunks = scores ? 1 : (int)sv_chunks(A.cols, nkv, max_len);
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
