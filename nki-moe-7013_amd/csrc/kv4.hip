// The cache in 4 bits: a prompt's rows into it, a decode step's projection rows
// into it, and its values back (head_dim 128; the format is in kv4.hpp).
#include "attn_tile.hpp"
#include "kv4.hpp"

#include <math.h>

namespace qmoe {

// Rows go through in chunks of KS_ROWS of a (sequence, kv head), 16 lanes a row: lane
// p % 16 has 8 elements, 16 bytes in bf16 and 4 in codes, so that a wave's loads and
// stores are whole lines; all of a thread's loads are in flight at once.  Bound by memory:
// 512 + 136 bytes a (token, kv head), two prompts of 8192 (42 MB each way) 9.3 us to the
// cache and 8.7 back under a profiler, 16.6 for both among other calls, 5 TB/s; a lane a
// block, 32 bytes apart, took 29.6 us for both instead of 17.2.
constexpr int KS_UNROLL = 4, KS_ROWS = 16 * KS_UNROLL;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, true));
}
constexpr int DPP_XOR1 = 0xb1, DPP_XOR2 = 0x4e;         // quad_perm [1,0,3,2], [2,3,0,1]
constexpr int DPP_ROR4 = 0x124, DPP_ROR8 = 0x128;       // row_ror

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
// Two bf16 values as numbers of the power's multiples (nearest, ties to even, what is
// past 6 to 6), to byte B of w.
template <int B>
__device__ __forceinline__ uint32_t kv4_pack(uint32_t w, uint32_t x, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x), scale, B);
}

__global__ __launch_bounds__(256) void kv4_store_kernel(
    const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int chunks, int n, int S_src,
    const int32_t* __restrict__ starts, const int32_t* __restrict__ lengths, int Hkv, int S_max,
    uint8_t* __restrict__ k4, uint8_t* __restrict__ ks, uint8_t* __restrict__ v4, uint8_t* __restrict__ vs) {
  const int bh = int(blockIdx.x) / chunks, b = bh / Hkv, p = threadIdx.x & 15;
  const int s0 = int(blockIdx.x) % chunks * KS_ROWS + int(threadIdx.x) / 16;
  const int len = lengths ? min(lengths[b], n) : n;
  const int64_t start = starts ? starts[b] : 0;
  const uint16_t* src = (blockIdx.y ? v : k) + int64_t(bh) * S_src * HD + p * 8;
  u32x4 x[KS_UNROLL];
#pragma unroll
  for (int u = 0; u < KS_UNROLL; ++u) {
    const int s = s0 + 16 * u;
    x[u] = s < len ? ld16(src + int64_t(s) * HD) : u32x4{0u, 0u, 0u, 0u};
  }
  uint8_t* codes = (blockIdx.y ? v4 : k4) + int64_t(bh) * S_max * KV4_ROWB + p * 4;
  uint32_t* powers = reinterpret_cast<uint32_t*>((blockIdx.y ? vs : ks) + int64_t(bh) * S_max * 4);
#pragma unroll
  for (int u = 0; u < KS_UNROLL; ++u) {
    // the block's largest magnitude, over its four lanes: bf16's bits without the sign
    // are in the order of the magnitudes
    uint32_t top = pk_max(pk_max(x[u].x & 0x7fff7fffu, x[u].y & 0x7fff7fffu),
                          pk_max(x[u].z & 0x7fff7fffu, x[u].w & 0x7fff7fffu));
    top = pk_max(top, dpp_u32<DPP_XOR1>(top));
    top = pk_max(top, dpp_u32<DPP_XOR2>(top));
    const int power = kv4_power(kv4_wants(__uint_as_float(max(top << 16, top & 0xffff0000u))));
    const float scale = kv4_scale(uint32_t(power));
    uint32_t c = kv4_pack<0>(0u, x[u].x, scale);
    c = kv4_pack<1>(c, x[u].y, scale);
    c = kv4_pack<2>(c, x[u].z, scale);
    c = kv4_pack<3>(c, x[u].w, scale);
    uint32_t all = uint32_t(power) << (8 * (p >> 2));  // the row's four powers
    all |= dpp_u32<DPP_ROR4>(all);
    all |= dpp_u32<DPP_ROR8>(all);
    const int s = s0 + 16 * u;
    const int64_t to = start + s;
    if (s < len && to >= 0 && to < S_max) {
      *reinterpret_cast<uint32_t*>(codes + to * KV4_ROWB) = power == KV4_NAN ? 0u : c;
      if (p == 0) powers[to] = all;
    }
  }
}

__global__ __launch_bounds__(256) void kv4_load_kernel(
    const uint8_t* __restrict__ k4, const uint8_t* __restrict__ ks, const uint8_t* __restrict__ v4,
    const uint8_t* __restrict__ vs, int chunks, int n, int S_max, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
  const int bh = int(blockIdx.x) / chunks, p = threadIdx.x & 15;
  const int s0 = int(blockIdx.x) % chunks * KS_ROWS + int(threadIdx.x) / 16;
  const uint8_t* codes = (blockIdx.y ? v4 : k4) + int64_t(bh) * S_max * KV4_ROWB + p * 4;
  const uint8_t* powers = (blockIdx.y ? vs : ks) + int64_t(bh) * S_max * 4 + (p >> 2);
  uint16_t* dst = (blockIdx.y ? v : k) + int64_t(bh) * n * HD + p * 8;
  uint32_t w[KS_UNROLL], power[KS_UNROLL];
#pragma unroll
  for (int u = 0; u < KS_UNROLL; ++u) {
    const int s = min(s0 + 16 * u, n - 1);
    w[u] = *reinterpret_cast<const uint32_t*>(codes + int64_t(s) * KV4_ROWB);
    power[u] = powers[int64_t(s) * 4];
  }
#pragma unroll
  for (int u = 0; u < KS_UNROLL; ++u) {
    const float scale = kv4_scale(power[u]);
    if (s0 + 16 * u < n)
      *reinterpret_cast<u32x4*>(dst + int64_t(s0 + 16 * u) * HD) = u32x4{
          kv4_pair<0>(w[u], scale), kv4_pair<1>(w[u], scale), kv4_pair<2>(w[u], scale), kv4_pair<3>(w[u], scale)};
  }
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

// Bound by latency: one launch, one round trip for the row and one for the tables at its
// position (1 row 3.2 us, 64 rows 3.9; 20 KB of the projection a row of 40 heads).
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
  QMOE_REQUIRE((reinterpret_cast<uintptr_t>(k_scales) | reinterpret_cast<uintptr_t>(v_scales)) % 4 == 0,
               "%s: scales must be 4-byte aligned", fn);
  const int64_t chunks = (n + KS_ROWS - 1) / KS_ROWS;
  QMOE_REQUIRE(B * Hkv * chunks < (1ll << 31), "%s: grid too large", fn);
  hipLaunchKernelGGL(kv4_store_kernel, dim3(unsigned(B * Hkv * chunks), 2), dim3(256), 0, as_stream(stream), k, v,
                     int(chunks), int(n), int(S_src), starts, lengths, int(Hkv), int(S_max), k_cache, k_scales, v_cache,
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
  const int64_t chunks = (n + KS_ROWS - 1) / KS_ROWS;
  QMOE_REQUIRE(B * Hkv * chunks < (1ll << 31), "%s: grid too large", fn);
  hipLaunchKernelGGL(kv4_load_kernel, dim3(unsigned(B * Hkv * chunks), 2), dim3(256), 0, as_stream(stream), k_cache,
                     k_scales, v_cache, v_scales, int(chunks), int(n), int(S_max), k, v);
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
