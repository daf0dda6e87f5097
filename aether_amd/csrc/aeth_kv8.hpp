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

// bytes i of four words as one word for each i: r[i] = {a.i, b.i, c.i, d.i}
__device__ __forceinline__ void kv8_transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&r)[4]) {
    const uint32_t p = __builtin_amdgcn_perm(b, a, 0x05010400u), q = __builtin_amdgcn_perm(d, c, 0x05010400u);
    const uint32_t s = __builtin_amdgcn_perm(b, a, 0x07030602u), t = __builtin_amdgcn_perm(d, c, 0x07030602u);
    r[0] = __builtin_amdgcn_perm(q, p, 0x05040100u);
    r[1] = __builtin_amdgcn_perm(q, p, 0x07060302u);
    r[2] = __builtin_amdgcn_perm(t, s, 0x05040100u);
    r[3] = __builtin_amdgcn_perm(t, s, 0x07060302u);
}
