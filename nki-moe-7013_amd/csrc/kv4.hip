// The cache in 4 bits: a prompt's rows into it, a decode step's projection rows
// into it, and its values back (head_dim 128; the format is in kv4.hpp).
#include "attn_tile.hpp"
#include "kv4.hpp"

#include <math.h>

namespace qmoe {

// One thread a block of 32 elements: 64 bytes in, 16 bytes and a power out.
__global__ __launch_bounds__(256) void kv4_store_kernel(
    const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int64_t blocks, int n, int S_src,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lengths, int Hkv, int S_max,
    uint8_t* __restrict__ k4, uint8_t* __restrict__ ks, uint8_t* __restrict__ v4, uint8_t* __restrict__ vs) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= blocks) return;
  const int blk = int(i & 3);
  const int64_t r = i >> 2;  // (b, kv head, token)
  const int s = int(r % n);
  const int64_t bh = r / n;
  const int b = int(bh / Hkv);
  const int64_t to = int64_t(starts ? starts[b] : 0) + s;
  if (s >= (lengths ? lengths[b] : n) || to < 0 || to >= S_max) return;
  const uint16_t* src = (blockIdx.y ? v : k) + (bh * S_src + s) * HD + blk * KV4_BLOCK;
  float x[KV4_BLOCK];
  int wants = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const u32x4 w = ld16(src + c * 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[c * 8 + 2 * e] = bf16_lo(w[e]);
      x[c * 8 + 2 * e + 1] = bf16_hi(w[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < KV4_BLOCK; ++e) wants = max(wants, kv4_wants(x[e]));
  const int power = kv4_power(wants);
  u32x4 out;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= kv4_code(x[c * 8 + e], power) << (4 * e);
    out[c] = w;
  }
  const int64_t at = bh * S_max + to;
  *reinterpret_cast<u32x4*>((blockIdx.y ? v4 : k4) + at * KV4_ROWB + blk * 16) = out;
  (blockIdx.y ? vs : ks)[at * 4 + blk] = uint8_t(power);
}

// One thread a block of 32 elements: 16 bytes and a power in, 64 bytes out.
__global__ __launch_bounds__(256) void kv4_load_kernel(
    const uint8_t* __restrict__ k4, const uint8_t* __restrict__ ks, const uint8_t* __restrict__ v4,
    const uint8_t* __restrict__ vs, int64_t blocks, int n, int S_max, uint16_t* __restrict__ k,
    uint16_t* __restrict__ v) {
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= blocks) return;
  const int blk = int(i & 3);
  const int64_t r = i >> 2, at = r / n * S_max + r % n;
  const u32x4 w = ld16((blockIdx.y ? v4 : k4) + at * KV4_ROWB + blk * 16);
  const float scale = kv4_scale((blockIdx.y ? vs : ks)[at * 4 + blk]);
  uint16_t* dst = (blockIdx.y ? v : k) + r * HD + blk * KV4_BLOCK;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<u32x4*>(dst + c * 8) = u32x4{kv4_pair<0>(w[c], scale), kv4_pair<1>(w[c], scale),
                                                   kv4_pair<2>(w[c], scale), kv4_pair<3>(w[c], scale)};
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m, 64);
  return v;
}
__device__ __forceinline__ int half_max(int v) {
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) v = max(v, __shfl_xor(v, m, 64));
  return v;
}

// Half an entry into the cache: lane l holds element l of the 64 from `half` on.
template <class T>
__device__ __forceinline__ void kv4_put(uint8_t* codes, uint8_t* powers, int half, int l, T x) {
  const int power = kv4_power(half_max(kv4_wants(x)));
  uint32_t c = kv4_code(x, power);
  c |= uint32_t(__shfl_down(int(c), 1, 64)) << 4;  // of even lanes: a byte
  c |= uint32_t(__shfl_down(int(c), 2, 64)) << 8;
  c |= uint32_t(__shfl_down(int(c), 4, 64)) << 16;
  if (l % 8 == 0) *reinterpret_cast<uint32_t*>(codes + half * 32 + l / 2) = c;
  if (l % 32 == 0) powers[half * 2 + l / 32] = uint8_t(power);
}

// One wave a (head, token): lane l holds elements l and l + 64, which RoPE pairs.
// Queries are computed in 32 bits, as in kv_append; keys in 64, because a key next
// to the border of two numbers is half a number off if it lands on the wrong side
// (32 bits put about one of 3 million elements there), and they are few.
__global__ __launch_bounds__(64) void kv4_append_kernel(
    const float* __restrict__ raw, const uint16_t* __restrict__ qn_w, const uint16_t* __restrict__ kn_w,
    const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, const int32_t* __restrict__ positions,
    const int32_t* __restrict__ slots, int S, int Hq, int Hkv, int S_max, int max_pos, float eps,
    uint16_t* __restrict__ q_out, uint8_t* __restrict__ k4, uint8_t* __restrict__ ks, uint8_t* __restrict__ v4,
    uint8_t* __restrict__ vs) {
  const int l = threadIdx.x, head = blockIdx.x, t = blockIdx.y;
  const float* p = raw + (int64_t(t) * (Hq + 2 * Hkv) + head) * HD;
  float lo = p[l], hi = p[l + 64];
  const int pos = positions[t], slot = slots[t];
  const bool ok = pos >= 0 && pos < max_pos && slot >= 0 && slot < S_max;
  if (!ok && head >= Hq) return;  // a rejected row: no entry, q zero
  const int kvh = (head - Hq) % Hkv;
  const int64_t at = (int64_t(t / S) * Hkv + kvh) * S_max + slot;
  if (head >= Hq + Hkv) {
    kv4_put(v4 + at * KV4_ROWB, vs + at * 4, 0, l, lo);
    kv4_put(v4 + at * KV4_ROWB, vs + at * 4, 1, l, hi);
    return;
  }
  const uint16_t* nw = head < Hq ? qn_w : kn_w;
  const float wl = bf16_to_f32(nw[l]), wh = bf16_to_f32(nw[l + 64]);
  const int64_t rope = int64_t(ok ? pos : 0) * (HD / 2) + l;
  const float c = rope_cos[rope], sn = rope_sin[rope];
  if (head < Hq) {
    const float r = rsqrtf(wave_sum(lo * lo + hi * hi) / float(HD) + eps);
    const float x = wl * (lo * r), y = wh * (hi * r);
    uint16_t* dst = q_out + (int64_t(t) * Hq + head) * HD;
    dst[l] = f32_to_bf16(ok ? x * c - y * sn : 0.0f);
    dst[l + 64] = f32_to_bf16(ok ? y * c + x * sn : 0.0f);
    return;
  }
  const double dl = lo, dh = hi;
  const double r = 1.0 / sqrt(wave_sum64(dl * dl + dh * dh) / double(HD) + double(eps));
  const double x = dl * r * double(wl), y = dh * r * double(wh);
  kv4_put(k4 + at * KV4_ROWB, ks + at * 4, 0, l, x * double(c) - y * double(sn));
  kv4_put(k4 + at * KV4_ROWB, ks + at * 4, 1, l, y * double(c) + x * double(sn));
}

}  // namespace qmoe

using namespace qmoe;

static int kv4_check(const char* fn, int64_t B, int64_t Hkv, int64_t D, int64_t S_max, int64_t n) {
  QMOE_REQUIRE(D == HD, "%s: head_dim must be 128 (D=%lld)", fn, (long long)D);
  QMOE_REQUIRE(B >= 0 && B < 65536 && Hkv > 0 && Hkv < 65536 && S_max > 0 && S_max < (1ll << 30),
               "%s: bad B/Hkv/S_max", fn);
  QMOE_REQUIRE(n >= 0 && n < (1ll << 30) && B * Hkv * n < (1ll << 36), "%s: bad number of entries", fn);
  return QMOE_OK;
}

extern "C" int qmoe_kv4_store(const qmoe_bf16* k, const qmoe_bf16* v, int64_t S_src, int64_t n, const int32_t* starts,
                              const int32_t* lengths, int64_t B, int64_t Hkv, int64_t D, int64_t S_max,
                              uint8_t* k_cache, uint8_t* k_scales, uint8_t* v_cache, uint8_t* v_scales,
                              qmoe_stream_t stream) {
  const char* fn = "qmoe_kv4_store";
  QMOE_REQUIRE(B == 0 || n == 0 || (k && v && k_cache && k_scales && v_cache && v_scales), "%s: null pointer", fn);
  if (int rc = kv4_check(fn, B, Hkv, D, S_max, n)) return rc;
  QMOE_REQUIRE(S_src >= n && S_src < (1ll << 30), "%s: need n <= S_src", fn);
  if (B == 0 || n == 0) return QMOE_OK;
  QMOE_REQUIRE(aligned16(k, v, k_cache, v_cache), "%s: operands must be 16-byte aligned", fn);
  const int64_t blocks = B * Hkv * n * 4;
  hipLaunchKernelGGL(kv4_store_kernel, dim3(unsigned((blocks + 255) / 256), 2), dim3(256), 0, as_stream(stream), k, v,
                     blocks, int(n), int(S_src), starts, lengths, int(Hkv), int(S_max), k_cache, k_scales, v_cache,
                     v_scales);
  return hip_status(fn);
}

extern "C" int qmoe_kv4_load(const uint8_t* k_cache, const uint8_t* k_scales, const uint8_t* v_cache,
                             const uint8_t* v_scales, int64_t B, int64_t Hkv, int64_t D, int64_t S_max, int64_t n,
                             qmoe_bf16* k, qmoe_bf16* v, qmoe_stream_t stream) {
  const char* fn = "qmoe_kv4_load";
  QMOE_REQUIRE(B == 0 || n == 0 || (k && v && k_cache && k_scales && v_cache && v_scales), "%s: null pointer", fn);
  if (int rc = kv4_check(fn, B, Hkv, D, S_max, n)) return rc;
  QMOE_REQUIRE(n <= S_max, "%s: need n <= S_max", fn);
  if (B == 0 || n == 0) return QMOE_OK;
  QMOE_REQUIRE(aligned16(k, v, k_cache, v_cache), "%s: operands must be 16-byte aligned", fn);
  const int64_t blocks = B * Hkv * n * 4;
  hipLaunchKernelGGL(kv4_load_kernel, dim3(unsigned((blocks + 255) / 256), 2), dim3(256), 0, as_stream(stream),
                     k_cache, k_scales, v_cache, v_scales, blocks, int(n), int(S_max), k, v);
  return hip_status(fn);
}

extern "C" int qmoe_kv4_append(const float* qkv, const qmoe_bf16* q_norm_w, const qmoe_bf16* k_norm_w,
                               const float* rope_cos, const float* rope_sin, int64_t max_pos,
                               const int32_t* positions, const int32_t* slots, int64_t B, int64_t S, int64_t Hq,
                               int64_t Hkv, int64_t D, int64_t S_max, float eps, qmoe_bf16* q_out, uint8_t* k_cache,
                               uint8_t* k_scales, uint8_t* v_cache, uint8_t* v_scales, qmoe_stream_t stream) {
  const char* fn = "qmoe_kv4_append";
  QMOE_REQUIRE(q_norm_w && k_norm_w && rope_cos && rope_sin &&
                   (B == 0 || S == 0 || (qkv && positions && slots && q_out && k_cache && k_scales && v_cache && v_scales)),
               "%s: null pointer", fn);
  if (int rc = kv4_check(fn, B, Hkv, D, S_max, 0)) return rc;
  QMOE_REQUIRE(Hq > 0 && Hq % Hkv == 0 && Hq < 65536 && Hq + 2 * Hkv < 65536, "%s: bad head counts", fn);
  QMOE_REQUIRE(S >= 0 && S < 65536 && B * S < 65536, "%s: B * S must be below 65536", fn);
  QMOE_REQUIRE(max_pos > 0, "%s: bad max_pos", fn);
  if (B == 0 || S == 0) return QMOE_OK;
  QMOE_REQUIRE(reinterpret_cast<uintptr_t>(k_cache) % 4 == 0 && reinterpret_cast<uintptr_t>(v_cache) % 4 == 0,
               "%s: caches must be 4-byte aligned", fn);
  hipLaunchKernelGGL(kv4_append_kernel, dim3(unsigned(Hq + 2 * Hkv), unsigned(B * S)), dim3(64), 0, as_stream(stream),
                     qkv, q_norm_w, k_norm_w, rope_cos, rope_sin, positions, slots, int(S), int(Hq), int(Hkv),
                     int(S_max), int(std::min<int64_t>(max_pos, 1ll << 30)), eps, q_out, k_cache, k_scales, v_cache,
                     v_scales);
  return hip_status(fn);
}
