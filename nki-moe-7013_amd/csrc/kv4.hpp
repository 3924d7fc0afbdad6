// Entries of the 4-bit cache (head_dim 128).
//
// An entry is 128 e2m1 numbers, two a byte with the even element in the low half,
// and a power of two (a byte p for 2^(p - 127)) for every 32 of them: the block
// format that gfx950's conversions take, 68 bytes where bf16 takes 256.  The
// power is the smallest whose seventh multiple is above the block's largest
// magnitude (6 is the largest number, and up to 7 it is the nearest one), so it
// hangs on the largest element alone: its exponent, one more where its mantissa is
// 1.75 or more, less 2.  A block with an infinity or a NaN has the power 255 and
// reads as NaN.
#pragma once

#include "attn_tile.hpp"
#include "common.hpp"

namespace qmoe {

constexpr int KV4_ROWB = 64;    // bytes of an entry's numbers
constexpr int KV4_BLOCK = 32;   // elements that share a power
constexpr int KV4_NAN = 255;
constexpr int KV4_LOW = 7, KV4_HIGH = 252;  // powers of finite blocks: 6 * 2^125 is finite in bf16, 2^-120 / 2 normal

// The power's exponent that one element asks for (a block takes the largest),
// biased by 127 and not yet clamped.  Adding a quarter to the mantissa carries
// into the exponent from 1.75 on.
constexpr int KV4_NONFINITE = 1 << 16;
__device__ __forceinline__ int kv4_wants(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u >= 0x7f800000u ? KV4_NONFINITE : int((u + (1u << 21)) >> 23) - 2;
}
__device__ __forceinline__ int kv4_wants(double x) {
  const uint64_t u = uint64_t(__double_as_longlong(x)) & 0x7fffffffffffffffull;
  return u >= 0x7ff0000000000000ull ? KV4_NONFINITE : int((u + (1ull << 50)) >> 52) - (1023 - 127) - 2;
}
__device__ __forceinline__ int kv4_power(int wants) {
  return wants == KV4_NONFINITE ? KV4_NAN : min(max(wants, KV4_LOW), KV4_HIGH);
}

__device__ __forceinline__ float kv4_inverse(float, int power) { return __uint_as_float(uint32_t(254 - power) << 23); }
__device__ __forceinline__ double kv4_inverse(double, int power) {
  return __longlong_as_double(int64_t(1023 + 127 - power) << 52);
}

// The nearest e2m1 number of x / 2^(power - 127), ties to the even code, with x's
// sign.  The division is exact, so the result is that of the real number x.
__device__ __forceinline__ uint32_t kv4_sign(float x) { return __float_as_uint(x) >> 28 & 8u; }
__device__ __forceinline__ uint32_t kv4_sign(double x) { return uint32_t(uint64_t(__double_as_longlong(x)) >> 60) & 8u; }
template <class T>
__device__ __forceinline__ uint32_t kv4_code(T x, int power) {
  if (power == KV4_NAN) return 0;
  const T y = fabs(x) * kv4_inverse(x, power);
  const uint32_t n = uint32_t(y > T(0.25)) + uint32_t(y >= T(0.75)) + uint32_t(y > T(1.25)) + uint32_t(y >= T(1.75)) +
                     uint32_t(y > T(2.5)) + uint32_t(y >= T(3.5)) + uint32_t(y > T(5.0));
  return n | kv4_sign(x);
}

// The multiplier of a block's numbers: 2^(power - 127), NaN for 255.
__device__ __forceinline__ float kv4_scale(uint32_t power) {
  return __uint_as_float(power == KV4_NAN ? 0x7fc00000u : power << 23);
}

// Two numbers of a byte times the block's multiplier, in bf16 (exact): byte `B` of w.
template <int B>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}

// 32 numbers of a block times its multiplier, as the four 16-byte chunks of a bf16 row.
__device__ __forceinline__ void kv4_chunks(const u32x4& w, float scale, u32x4 (&c)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    c[i] = u32x4{kv4_pair<0>(w[i], scale), kv4_pair<1>(w[i], scale), kv4_pair<2>(w[i], scale), kv4_pair<3>(w[i], scale)};
}

// Loads through a buffer resource: a word past its end is zero.
__device__ __forceinline__ u32x4 kv4_ld16(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, int(off), 0, 0));
}
__device__ __forceinline__ uint32_t kv4_ld1(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b8(r, int(off), 0, 0);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv4_rsrc(const uint8_t* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p), 0, int(bytes), 0x00020000);
}

// Tiles of 64 keys of a cache in 4 bits for flash_tiles: a thread holds a block of the
// next K and of the next V tile in registers, where their loads land during a step;
// load_k and load_v write a tile's blocks to LDS in bf16 and request the next
// tile's.  Calls go through the tiles in order.
struct Tiles4 {
  __amdgpu_buffer_rsrc_t rk, rks, rv, rvs;
  u32x4 kw, vw;
  uint32_t kp, vp;
  int key, n_kt, row, blk;
  uint8_t* smem;
  Gap g;
  // rows: rows of the cache that the run may touch
  __device__ __forceinline__ void start(uint8_t* lds, const uint8_t* k, const uint8_t* ks, const uint8_t* v,
                                        const uint8_t* vs, int rows, int k0, int tiles, Gap gap) {
    rk = kv4_rsrc(k, int64_t(rows) * KV4_ROWB);
    rv = kv4_rsrc(v, int64_t(rows) * KV4_ROWB);
    rks = kv4_rsrc(ks, int64_t(rows) * 4);
    rvs = kv4_rsrc(vs, int64_t(rows) * 4);
    smem = lds;
    // rows 2 apart next to each other: eight lanes' chunks, of K as of V, then lie in
    // eight places
    const int q = int(threadIdx.x) >> 2;
    row = (q & ~3) | (q & 1) << 1 | ((q >> 1) & 1);
    blk = int(threadIdx.x) & 3;
    key = k0 + row;
    n_kt = tiles;
    g = gap;
    fetch_k(0);
    fetch_v(0);
  }
  __device__ __forceinline__ void fetch_k(int kt) {
    const uint32_t r = uint32_t(g.row(key + kt * AP_KT));
    kw = kv4_ld16(rk, r * KV4_ROWB + blk * 16);
    kp = kv4_ld1(rks, r * 4 + blk);
  }
  __device__ __forceinline__ void fetch_v(int kt) {
    const uint32_t r = uint32_t(g.row(key + kt * AP_KT));
    vw = kv4_ld16(rv, r * KV4_ROWB + blk * 16);
    vp = kv4_ld1(rvs, r * 4 + blk);
  }
  __device__ __forceinline__ void load_k(int kt, int buf) {
    u32x4 c[4];
    kv4_chunks(kw, kv4_scale(kp), c);
    uint8_t* to = smem + buf * AP_TILE + row * AP_ROWB;
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(to + ap_kslot(row, 4 * blk + i) * 16) = c[i];
    if (kt + 1 < n_kt) fetch_k(kt + 1);
  }
  __device__ __forceinline__ void load_v(int kt, int buf) {
    u32x4 c[4];
    kv4_chunks(vw, kv4_scale(vp), c);
    uint8_t* to = smem + (2 + buf) * AP_TILE + row * AP_ROWB;
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(to + ap_vslot(row, 4 * blk + i) * 16) = c[i];
    if (kt + 1 < n_kt) fetch_v(kt + 1);
  }
  __device__ __forceinline__ void landed_but_one() const {}
  __device__ __forceinline__ void landed() const {}
};

// Keys [k0, k1) (k0 < k1) of a window's run over a cache in 4 bits.
__device__ __forceinline__ void flash_segment(uint8_t* smem, const uint8_t* k, const uint8_t* ks, const uint8_t* v,
                                              const uint8_t* vs, int k0, int k1, const Windowed& see,
                                              float scale_log2, FlashRows& st) {
  Tiles4 tiles;
  const int n_kt = (k1 - k0 + AP_KT - 1) / AP_KT;
  tiles.start(smem, k, ks, v, vs, see.g.row(k1 - 1) + 1, k0, n_kt, see.g);
  flash_tiles(smem, tiles, n_kt, k0, see, scale_log2, st);
}

}  // namespace qmoe
