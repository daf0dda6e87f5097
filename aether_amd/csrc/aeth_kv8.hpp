// The 8-bit key/value cache of one layer and sequence: [kv_heads][tiles] tiles of
// 64 tokens, a tile being
//   K codes  int8 [64][hd]
//   V codes  int8 [hd][64], token t at byte aeth_kv8_vbyte(t) of a row
//   K scales f32 [64], V scales f32 [64]
// and a value code · scale. Tiles are contiguous, so a wave that takes one reads
// one run of 128·hd + 512 bytes. Both code planes are int8 matrix operands as they
// stand (v_mfma_i32_16x16x64_i8, lane l: row l%16, bytes 16·(l/16) ..): K's rows are
// the scores' rows; a row of V is one output dimension over the tile's tokens, in
// the order in which the scores of four 16-token products stand in a lane's
// registers (lane group g = l/16 holds tokens 16j + 4g + r, j and r = 0 .. 3), so
// that the probabilities are the other operand without leaving their lane.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define KV8_TILE 64

__host__ __device__ constexpr int64_t aeth_kv8_tile_bytes(int hd) { return 2 * KV8_TILE * (int64_t)hd + 8 * KV8_TILE; }
__host__ __device__ constexpr int aeth_kv8_vbyte(int t) { return 16 * ((t >> 2) & 3) + 4 * (t >> 4) + (t & 3); }
// the longest cache: positions stay within int32 with a tile and a window to spare
constexpr int64_t KV8_MAX_SEQ = (int64_t)1 << 30;
inline bool aeth_kv8_head_dim(int64_t hd) { return hd == 64 || hd == 128 || hd == 256; }

// A rotated pair (apply_rope_inplace, runner.rs:1886-1909), rounded as k_rope's is: a head without a norm gets aeth_rope's bits
__device__ __forceinline__ float kv8_rot0(float a, float b, float sn, float cs) { return fmaf(a, cs, -(b * sn)); }
__device__ __forceinline__ float kv8_rot1(float a, float b, float sn, float cs) { return fmaf(a, sn, b * cs); }
__device__ __forceinline__ void kv8_rotate(float4& a, float4& b, float4 sn, float4 cs) {
    const float4 x = a, y = b;
    a = make_float4(kv8_rot0(x.x, y.x, sn.x, cs.x), kv8_rot0(x.y, y.y, sn.y, cs.y), kv8_rot0(x.z, y.z, sn.z, cs.z), kv8_rot0(x.w, y.w, sn.w, cs.w));
    b = make_float4(kv8_rot1(x.x, y.x, sn.x, cs.x), kv8_rot1(x.y, y.y, sn.y, cs.y), kv8_rot1(x.z, y.z, sn.z, cs.z), kv8_rot1(x.w, y.w, sn.w, cs.w));
}

// ── quantising: codes 127·x / amax to the nearest integer, ties to even, of the exact quotient ──
template <int L>
__device__ __forceinline__ uint32_t kv8_umax(uint32_t v) {  // max over aligned groups of L lanes (8, 16 or 32)
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, false));
    if (L >= 16) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xF, 0xF, false));
    if (L >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(a[0], a[1]);
    }
    return v;
}

__device__ __forceinline__ uint32_t kv8_abs_max(uint32_t m, float4 y) {  // as integers: a NaN's bits are above an infinity's
    m = max(max(m, __float_as_uint(y.x) & 0x7FFFFFFFu), __float_as_uint(y.y) & 0x7FFFFFFFu);
    return max(max(m, __float_as_uint(y.z) & 0x7FFFFFFFu), __float_as_uint(y.w) & 0x7FFFFFFFu);
}

// 127 / amax in f64 to 2^-50 relative (amax > 0), by two Newton steps on the reciprocal instruction
__device__ __forceinline__ double kv8_inverse(float amax) {
    const double a = (double)amax;
    double r = __builtin_amdgcn_rcp(a);
    r = fma(fma(-a, r, 1.0), r, r);
    r = fma(fma(-a, r, 1.0), r, r);
    return 127.0 * r;
}

// rint(127·x / amax): with amax = A·2^a, A below 2^24, and x = X·2^(a - s) a tie's distance |127·X / (A·2^s) - (i + 1/2)| is 0 or at
// least 1 / (A·2^max(s, 1)). Quotients of a half and more have s up to 8: 2^-32 (smaller ones are far from a tie). So the f64
// product (off by under 2^-42) rounded to a multiple of 2^-40 is a tie exactly where the quotient is.
__device__ __forceinline__ uint32_t kv8_code(float x, double inv) {
    const double t = (double)x * inv;
    const double u = (t + 6144.0) - 6144.0;
    return (uint32_t)__double2loint(u + 6755399441055744.0) & 0xFFu;  // 1.5·2^52
}

__device__ __forceinline__ uint32_t kv8_code4(float4 y, double inv, bool finite) {
    const uint32_t w = kv8_code(y.x, inv) | kv8_code(y.y, inv) << 8 | kv8_code(y.z, inv) << 16 | kv8_code(y.w, inv) << 24;
    return finite ? w : 0;
}

// The codes and the scale of a row whose dimensions e .. e + 3 (a) and hd/2 further on (b) a lane holds, hd/8 lanes a row.
// Every lane of the wave has to call it.
struct Kv8Row {
    uint32_t a, b;
    float scale;
};
template <int HD>
__device__ __forceinline__ Kv8Row kv8_quantise(float4 a, float4 b) {
    const uint32_t m = kv8_umax<HD / 8>(kv8_abs_max(kv8_abs_max(0, a), b));
    const bool finite = m < 0x7F800000u;
    const float amax = __uint_as_float(m);
    const double inv = finite && m > 0 ? kv8_inverse(amax) : 0.0;
    return {kv8_code4(a, inv, finite), kv8_code4(b, inv, finite), finite ? amax / 127.0f : __uint_as_float(0x7FC00000u)};
}
// ... into slot `slot` of a head's tiles, as K (v = 0) or V (1)
template <int HD>
__device__ __forceinline__ void kv8_put(uint8_t* tiles, int64_t slot, int v, int e, const Kv8Row& q) {
    const int t = (int)(slot & 63);
    uint8_t* base = tiles + (slot >> 6) * aeth_kv8_tile_bytes(HD);
    if (v) {
        uint8_t* dst = base + KV8_TILE * HD + e * KV8_TILE + aeth_kv8_vbyte(t);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            dst[i * KV8_TILE] = (uint8_t)(q.a >> (8 * i));
            dst[(HD / 2 + i) * KV8_TILE] = (uint8_t)(q.b >> (8 * i));
        }
    } else {
        *(uint32_t*)(base + t * HD + e) = q.a;
        *(uint32_t*)(base + t * HD + HD / 2 + e) = q.b;
    }
    if (e == 0) *(float*)(base + 2 * KV8_TILE * HD + 4 * (KV8_TILE * v + t)) = q.scale;
}

// bytes i of four words as one word for each i: r[i] = {a.i, b.i, c.i, d.i}
__device__ __forceinline__ void kv8_transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&r)[4]) {
    const uint32_t p = __builtin_amdgcn_perm(b, a, 0x05010400u), q = __builtin_amdgcn_perm(d, c, 0x05010400u);
    const uint32_t s = __builtin_amdgcn_perm(b, a, 0x07030602u), t = __builtin_amdgcn_perm(d, c, 0x07030602u);
    r[0] = __builtin_amdgcn_perm(q, p, 0x05040100u);
    r[1] = __builtin_amdgcn_perm(q, p, 0x07060302u);
    r[2] = __builtin_amdgcn_perm(t, s, 0x05040100u);
    r[3] = __builtin_amdgcn_perm(t, s, 0x07060302u);
}
