// A key/value cache of bounded size that keeps the entries with the most
// accumulated attention weight (head_dim 128).
//
// Next to K and V [B][Hkv][S_max][D] the cache holds, for each slot of each kv
// head, the score (the attention weight that queries gave the entry, summed
// over queries and over the q heads of the group) and the token position.
// Keys are stored rotated, so the slots' order does not matter to attention and
// a kept entry may move to any free slot.
//
//  kv_append_kernel     raw projection -> normed, rotated q; K/V row, position
//                       and a zero score into a slot that need not be the
//                       position.
//  attn_scored_kernel   split-key decode attention that stores the scaled
//                       logits, and attn_scored_finish_kernel, which joins the
//                       splits and, now that a row's maximum and sum are known,
//                       adds 2^(s - m) / l to the scores.
//  kv_select_kernel     the kept entries of a (batch, kv head) by radix select.
//  kv_move_kernel       kept entries past the budget into the free slots below
//                       it: sources all past, destinations all below the
//                       budget, so the moves of a cache within itself neither
//                       overlap nor depend on their order.
#include "attn_tile.hpp"
#include "common.hpp"

#include <math.h>

namespace qmoe {

// ====================================================================== append
// One wave a (head, token): lane l holds elements l and l + 64, which RoPE pairs.
// v / sqrt(mean(v^2) + eps) * w, then the rotation by the position's (cos, sin).
// Bound by its one chain of memory round trips (1 row 2.5 us, 64 rows 2.9).
__global__ __launch_bounds__(64) void kv_append_kernel(
    const float* __restrict__ raw, const uint16_t* __restrict__ qn_w, const uint16_t* __restrict__ kn_w,
    const float* __restrict__ rope_cos, const float* __restrict__ rope_sin, const int32_t* __restrict__ positions,
    const int32_t* __restrict__ slots, int Hq, int Hkv, int S_max, int max_pos, float eps,
    uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_cache, uint16_t* __restrict__ v_cache,
    float* __restrict__ scores, int32_t* __restrict__ slot_pos) {
  const int l = threadIdx.x, head = blockIdx.x, b = blockIdx.y;
  const float* v = raw + (int64_t(b) * (Hq + 2 * Hkv) + head) * HD;
  float lo = v[l], hi = v[l + 64];
  const bool normed = head < Hq + Hkv;
  const uint16_t* nw = head < Hq ? qn_w : kn_w;
  const float wl = normed ? bf16_to_f32(nw[l]) : 0.0f, wh = normed ? bf16_to_f32(nw[l + 64]) : 0.0f;
  const int pos = positions[b], slot = slots[b];
  const bool ok = pos >= 0 && pos < max_pos && slot >= 0 && slot < S_max;
  if (!ok && head >= Hq) return;  // a rejected row: no cache row, q zero
  if (normed) {
    const int64_t at = int64_t(ok ? pos : 0) * (HD / 2) + l;
    const float c = rope_cos[at], sn = rope_sin[at];
    const float r = rsqrtf(wave_sum(lo * lo + hi * hi) / float(HD) + eps);
    const float x = wl * (lo * r), y = wh * (hi * r);
    lo = x * c - y * sn;
    hi = y * c + x * sn;
  }
  uint16_t* dst;
  if (head < Hq) {
    dst = q_out + (int64_t(b) * Hq + head) * HD;
    lo = ok ? lo : 0.0f;
    hi = ok ? hi : 0.0f;
  } else {
    const int kvh = (head - Hq) % Hkv;
    const int64_t at = (int64_t(b) * Hkv + kvh) * S_max + slot;
    dst = (head < Hq + Hkv ? k_cache : v_cache) + at * HD;
    if (l == 0 && head < Hq + Hkv) {
      if (scores) scores[at] = 0.0f;
      if (slot_pos) slot_pos[at] = pos;
    }
  }
  dst[l] = f32_to_bf16(lo);
  dst[l + 64] = f32_to_bf16(hi);
}

// ====================================================================== scored decode
constexpr int SD_KEYS = 64;       // keys of a wave
constexpr int SD_WAVES = 4;       // waves of a workgroup, at most; their runs are joined in LDS
constexpr int SD_SLICE = 256;     // keys whose scores a workgroup of the finish adds to
constexpr int SD_REC = HD + 4;    // LDS record of a wave: m, l, 2 pad, O[HD]
constexpr int SD_MAX_G = 16;
constexpr int SD_VCH = SD_KEYS * HD / 8 / 64;  // 16-byte V chunks of a lane

struct SdArgs {
  const uint16_t *q, *k, *v;
  const int32_t* ctx_len;
  int B, Hq, Hkv, S_max, max_ctx, split, nsplit, ldl;  // split: keys of a workgroup; ldl: logits of a row
  float scale_log2;
  float* ml;      // [B][Hq][nsplit][2]: a split's maximum and sum
  float* part;    // [B][Hq][nsplit][HD]: its unnormalised output
  float* logits;  // [B][Hq][ldl], in log2 units
  float* scores;  // [B][Hkv][S_max]
  uint16_t* out;
  int n_merge;  // workgroups of the finish that join rows; the rest add to the scores
};

__device__ __forceinline__ int sd_ctx(const SdArgs& a, int b) { return min(max(a.ctx_len[b], 0), a.max_ctx); }

// Workgroup = (split of WAVES x 64 keys, kv head, row), wave = 64 of its keys with
// the G q heads in the columns of S^T = K . Q^T and O^T = V^T . P^T.  Every load of
// a wave is in flight at once, so a wave costs one round trip to memory; K and
// V take turns in the wave's own LDS tile.  The logits leave as four
// consecutive keys a lane.  The weights are rounded to bf16 for the MFMA with V alone
// (half a step each; relative error of the outputs 0.0017 against 64 bits, with
// the output's own rounding); their sum l and what the scores get stay in 32 bits.
// Bound by memory: 32 rows of up to 4160 entries, 171 MB,
// in 39 us (4.4 TB/s); 44 us with K's A operands loaded straight from the cache, 32
// bytes of each of 32 rows an instruction.
// WAVES = 1 (few keys in all): K does go straight into its operands, since the
// round through LDS is longer than what whole rows save (one row of 1100: 8.4 us, 8.7
// with it), there is no join of four waves, which is two barriers longer, and the
// finish has no more records than it can take at once.
template <int WAVES>
__global__ __launch_bounds__(WAVES * 64) void attn_scored_kernel(const SdArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t vs[WAVES][AP_TILE];
  constexpr int SPLIT = WAVES * SD_KEYS;
  const int lane = threadIdx.x & 63, col = lane & 31, hi = lane >> 5;
  const int wave = WAVES > 1 ? __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)) : 0;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, G = a.Hq / a.Hkv;
  const int ctx = sd_ctx(a, b);
  if (split * SPLIT >= ctx) return;  // the finish knows which splits hold keys
  const int kw0 = split * SPLIT + wave * SD_KEYS, nk = min(SD_KEYS, ctx - kw0);
  float m = -INFINITY, l = 0.0f;
  f32x16 oacc[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) oacc[db] = f32x16{};
  if (nk > 0) {  // wave-uniform
    const int64_t base = (int64_t(b) * a.Hkv + kvh) * a.S_max + kw0;
    // ka[mb][ks]: one wave, the A operand itself; four waves, chunk lane + 64 (8 mb + ks) of
    // the tile, as V's (rows past nk repeat the last one, their p is 0)
    u32x4 ka[2][HD / 16], vr[SD_VCH], qb[HD / 16];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      const uint16_t* kp = a.k + (base + min(mb * 32 + col, nk - 1)) * HD + hi * 8;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) {
        if constexpr (WAVES == 1) {
          ka[mb][ks] = ld16(kp + ks * 16);
        } else {
          const int c = lane + 64 * (8 * mb + ks);
          ka[mb][ks] = ld16(a.k + (base + min(c >> 4, nk - 1)) * HD + (c & 15) * 8);
        }
      }
    }
    const uint16_t* qp = a.q + (int64_t(b) * a.Hq + kvh * G + min(col, G - 1)) * HD + hi * 8;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) qb[ks] = ld16(qp + ks * 16);
#pragma unroll
    for (int i = 0; i < SD_VCH; ++i) {
      const int c = lane + 64 * i;
      vr[i] = ld16(a.v + (base + min(c >> 4, nk - 1)) * HD + (c & 15) * 8);
    }
    uint8_t* vb = vs[wave];
    if constexpr (WAVES > 1) {
#pragma unroll
      for (int i = 0; i < SD_VCH; ++i) {
        const int c = lane + 64 * i, r = c >> 4;
        *reinterpret_cast<u32x4*>(vb + r * AP_ROWB + ap_kslot(r, c & 15) * 16) = ka[i >> 3][i & 7];
      }
      wave_lds_sync();
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
          ka[mb][ks] = *reinterpret_cast<const u32x4*>(vb + (mb * 32 + col) * AP_ROWB + ap_kslot(col, 2 * ks + hi) * 16);
      wave_lds_sync();
    }
    f32x16 sc[2];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      sc[mb] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        sc[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ka[mb][ks]),
                                                         __builtin_bit_cast(bf16x8, qb[ks]), sc[mb], 0, 0, 0);
    }
    // element e of block mb: key mb * 32 + 8 (e / 4) + 4 hi + e % 4
    float* lg = a.logits + (int64_t(b) * a.Hq + kvh * G + min(col, G - 1)) * a.ldl + kw0 + hi * 4;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int g4 = 0; g4 < 4; ++g4) {
#pragma unroll
        for (int e = g4 * 4; e < g4 * 4 + 4; ++e) {
          const int key = mb * 32 + (e >> 2) * 8 + hi * 4 + (e & 3);
          sc[mb][e] = key < nk ? sc[mb][e] * a.scale_log2 : -INFINITY;
          m = fmaxf(m, sc[mb][e]);
        }
        if (col < G)
          *reinterpret_cast<float4*>(lg + mb * 32 + g4 * 8) =
              make_float4(sc[mb][g4 * 4], sc[mb][g4 * 4 + 1], sc[mb][g4 * 4 + 2], sc[mb][g4 * 4 + 3]);
      }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float mb0 = m == -INFINITY ? 0.0f : m;
    uint32_t pk[2][8];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(sc[mb][2 * i] - mb0), p1 = __builtin_amdgcn_exp2f(sc[mb][2 * i + 1] - mb0);
        l += p0 + p1;
        const bf16x2_t pp = {static_cast<__bf16>(p0), static_cast<__bf16>(p1)};
        pk[mb][i] = __builtin_bit_cast(uint32_t, pp);
      }
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int i = 0; i < SD_VCH; ++i) {
      const int c = lane + 64 * i, r = c >> 4;
      *reinterpret_cast<u32x4*>(vb + r * AP_ROWB + ap_vslot(r, c & 15) * 16) = vr[i];
    }
    wave_lds_sync();
    const int vg = lane >> 4, ve = (lane >> 2) & 3, vq = lane & 3;
    const uint32_t vlane = uint32_t((4 * (vg >> 1) + ve) * AP_ROWB +
                                    (((2 * (vg & 1) + (vq >> 1)) ^ (2 * (ve >> 1))) * 16) + 8 * (vq & 1));
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const u32x4 pw = {pk[s >> 1][(s & 1) * 4], pk[s >> 1][(s & 1) * 4 + 1], pk[s >> 1][(s & 1) * 4 + 2],
                        pk[s >> 1][(s & 1) * 4 + 3]};
      const bf16x8 pb = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const uint32_t va = vlane + uint32_t(64 * (db ^ ve));
        const s16x4 v0 = lds_read_tr16(vb + va + (16 * s) * AP_ROWB);
        const s16x4 v1 = lds_read_tr16(vb + va + (16 * s + 8) * AP_ROWB);
        const bf16x8 av = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        oacc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(av, pb, oacc[db], 0, 0, 0);
      }
    }
  }
  const int64_t rec0 = (int64_t(b) * a.Hq + kvh * G) * a.nsplit + split;  // q head c's: c * nsplit further
  if constexpr (WAVES == 1) {
    if (col < G) {
      const int64_t at = rec0 + int64_t(col) * a.nsplit;
      float* pg = a.part + at * HD;
      if (hi == 0) *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(m, l);
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int e4 = 0; e4 < 4; ++e4)
          *reinterpret_cast<float4*>(pg + db * 32 + e4 * 8 + hi * 4) =
              make_float4(oacc[db][e4 * 4], oacc[db][e4 * 4 + 1], oacc[db][e4 * 4 + 2], oacc[db][e4 * 4 + 3]);
    }
    return;
  }
  // the waves' (m, l, O) joined in LDS (the V tiles are free)
  float* rec = reinterpret_cast<float*>(&vs[0][0]);
  static_assert(WAVES * SD_MAX_G * SD_REC * 4 <= WAVES * AP_TILE, "records fit the V tiles");
  __syncthreads();
  if (col < G) {
    float* pg = rec + (wave * SD_MAX_G + col) * SD_REC;
    if (hi == 0) {
      pg[0] = m;
      pg[1] = l;
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int e4 = 0; e4 < 4; ++e4)
        *reinterpret_cast<float4*>(pg + 4 + db * 32 + e4 * 8 + hi * 4) =
            make_float4(oacc[db][e4 * 4], oacc[db][e4 * 4 + 1], oacc[db][e4 * 4 + 2], oacc[db][e4 * 4 + 3]);
  }
  __syncthreads();
  for (int i = int(threadIdx.x); i < G * HD; i += WAVES * 64) {
    const int c = i / HD, d = i % HD;
    float M = -INFINITY, L = 0.0f, O = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) M = fmaxf(M, rec[(w * SD_MAX_G + c) * SD_REC]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float* r = rec + (w * SD_MAX_G + c) * SD_REC;
      const float wt = r[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(r[0] - M);
      L = fmaf(wt, r[1], L);
      O = fmaf(wt, r[4 + d], O);
    }
    const int64_t at = rec0 + int64_t(c) * a.nsplit;
    if (d == 0) *reinterpret_cast<float2*>(a.ml + at * 2) = make_float2(M, L);
    a.part[at * HD + d] = O;
  }
}

// Maximum and sum of a row's splits: lane i takes split i, i + 64, ...  Every
// workgroup of the finish reads them, so they lie apart from the outputs (one row
// of 131072: 106 us, 129 with each pair in front of its output).
__device__ __forceinline__ void sd_row(const float* rec, int live, int lane, float& M, float& L) {
  M = -INFINITY;
  L = 0.0f;
  for (int c = 0; c < live; c += 64) {
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (c + lane < live) ml = *reinterpret_cast<const float2*>(rec + int64_t(c + lane) * 2);
    const float m = fmaxf(M, wave_max(ml.x));
    const float mz = m == -INFINITY ? 0.0f : m;
    L = L * __builtin_amdgcn_exp2f(M - mz) + wave_sum(ml.y * __builtin_amdgcn_exp2f(ml.x - mz));
    M = m;
  }
}

// Workgroups [0, n_merge): a wave joins one (row, q head).  The rest: 256 keys of
// a (row, kv head), a thread a key, scores += sum over the group of 2^(s - m) / l.
// 32 rows of up to 4160: 7.5 us, of which the logits' 11 MB are about 3; one row of
// 1100, two round trips: 4.4.
__global__ __launch_bounds__(256) void attn_scored_finish_kernel(const SdArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, G = a.Hq / a.Hkv;
  if (int(blockIdx.x) < a.n_merge) {
    const int row = int(blockIdx.x) * 4 + wave;
    if (row >= a.B * a.Hq) return;
    const int live = (sd_ctx(a, row / a.Hq) + a.split - 1) / a.split;
    const float* p = a.part + int64_t(row) * a.nsplit * HD;
    const float* rec = a.ml + int64_t(row) * a.nsplit * 2;
    float M, L;
    sd_row(rec, live, lane, M, L);
    float o0 = 0.0f, o1 = 0.0f;
    for (int i0 = 0; i0 < live; i0 += 8) {
      float2 v[8];
      float w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = min(i0 + u, live - 1);
        v[u] = *reinterpret_cast<const float2*>(p + int64_t(i) * HD + lane * 2);
        w[u] = i0 + u < live ? rec[2 * i] : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float wt = w[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w[u] - M);
        o0 = fmaf(wt, v[u].x, o0);
        o1 = fmaf(wt, v[u].y, o1);
      }
    }
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    reinterpret_cast<uint32_t*>(a.out + int64_t(row) * HD)[lane] = pack_bf16x2(o0 * inv, o1 * inv);
    return;
  }
  __shared__ float sm[SD_MAX_G], si[SD_MAX_G];
  const int slices = (a.ldl + SD_SLICE - 1) / SD_SLICE, x = int(blockIdx.x) - a.n_merge, bh = x / slices, b = bh / a.Hkv;
  const int key = x % slices * SD_SLICE + int(threadIdx.x), ctx = sd_ctx(a, b);
  if (key - int(threadIdx.x) >= ctx) return;
  const int live = (ctx + a.split - 1) / a.split;
  const int row0 = b * a.Hq + bh % a.Hkv * G;
  for (int g = wave; g < G; g += 4) {
    float M, L;
    sd_row(a.ml + int64_t(row0 + g) * a.nsplit * 2, live, lane, M, L);
    if (lane == 0) {
      sm[g] = M;
      si[g] = L > 0.0f ? 1.0f / L : 0.0f;
    }
  }
  __syncthreads();
  if (key >= ctx) return;
  float sum = 0.0f;
  for (int g = 0; g < G; ++g)
    sum += __builtin_amdgcn_exp2f(a.logits[int64_t(row0 + g) * a.ldl + key] - sm[g]) * si[g];
  a.scores[int64_t(bh) * a.S_max + key] += sum;
}

// ====================================================================== eviction
constexpr int EV_THREADS = 1024;
constexpr int EV_WAVES = EV_THREADS / 64;
constexpr int EV_BINS = 2048;
constexpr int EV_LDS_KEYS = 32768;  // ranks held in LDS up to here (128 KB), else read again

struct EvArgs {
  const float* scores;
  const int32_t* slot_pos;
  const int32_t* ctx_len;
  int B, Hkv, S_max, budget, recent, sink, S_out, lds_keys;
  float* scores_out;
  int32_t* pos_out;
  int32_t* src;     // [B][Hkv][budget]: the slot whose entry slot i gets
  int32_t* movers;  // [B][Hkv][budget]: kept slots past the budget, ascending
};

// Scores as unsigned integers of the same order; -0 as 0, NaN above +inf.
__device__ __forceinline__ uint32_t ev_rank(float f) {
  if (f != f) return 0xfffffffeu;
  const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup a (row, kv head).  The budget-th largest rank by radix select
// (11 + 11 + 10 bits, a histogram in LDS each), where protected entries (the
// first `sink` positions and the `recent` last ones) rank above all; of the
// entries at the threshold the lowest slots stay.  Each wave owns a run of slots
// and numbers its holes (free slots below the budget) and movers (kept slots past
// it) with ballots; the hole of each rank takes the mover of that rank.
//
// Caches of up to 1024 R slots: what bounds it is its chain of round trips and
// barriers (8 rows of 4096 slots, 0.3 MB: 9.6 us), so every thread reads its R
// slots at once, before the length is known, and keeps them in registers; a
// histogram of its own for each pass needs no clearing between them; one wave
// looks for the bin while the others wait; movers leave their score and position
// in LDS, not only their slot.  `moves`: of a cache cut down in place by few
// entries the rows move here as well (64 rows of 1088 slots, 64 moves: 6.7 us; with a
// launch of their own, and the ranks in LDS, 11.3 + 4).
struct EvMove {
  uint16_t *k, *v;  // nullptr: kv_move_kernel does it
};

// Inclusive sums and the maximum over a wave's lanes by DPP (as wave_sum).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(1), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(2), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(4), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(8), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_BCAST15, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_BCAST31, 0xc, 0xf, false);
  return v;
}
__device__ __forceinline__ int wave_max_int(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(v, v, QMOE_DPP_ROW_SHR(1), 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, QMOE_DPP_ROW_SHR(2), 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, QMOE_DPP_ROW_SHR(4), 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, QMOE_DPP_ROW_SHR(8), 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, QMOE_DPP_ROW_BCAST15, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(v, v, QMOE_DPP_ROW_BCAST31, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(v, 63);
}
// The waves' values of red[EV_WAVES], by four wide reads, summed over the waves
// before `wave` (total: over all).
__device__ __forceinline__ int waves_before(const int* red, int wave, int& total) {
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < EV_WAVES / 4; ++i) {
    const int4 v = *reinterpret_cast<const int4*>(red + 4 * i);
    const int q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      total += q[j];
      before += 4 * i + j < wave ? q[j] : 0;
    }
  }
  return before;
}

template <int R>
__global__ __launch_bounds__(EV_THREADS) void kv_select_kernel(const EvArgs a, const EvMove mvd) {
  constexpr int MOVERS = R * 512;  // at most half of the slots move
  extern __shared__ __attribute__((aligned(16))) uint32_t ev_smem[];
  uint32_t* hist = ev_smem;                                // [3][EV_BINS], a lane's 32 (16) bins 64 apart, from the top
  int* red = reinterpret_cast<int*>(hist + 3 * EV_BINS);   // [3][EV_WAVES]
  int* sel = red + 3 * EV_WAVES;                           // [3][4]: bin, entries above it, entries in it
  int* m_slot = sel + 16;                                  // [MOVERS] by rank
  float* m_score = reinterpret_cast<float*>(m_slot + MOVERS);
  int* m_pos = reinterpret_cast<int*>(m_score + MOVERS);
  int* h_slot = m_pos + MOVERS;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int bh = blockIdx.x;
  const float* sc = a.scores + int64_t(bh) * a.S_max;
  const int32_t* sp = a.slot_pos + int64_t(bh) * a.S_max;
  float* so = a.scores_out + int64_t(bh) * a.S_out;
  int32_t* po = a.pos_out + int64_t(bh) * a.S_out;
  int32_t* src = a.src + int64_t(bh) * a.budget;
  const bool same = a.scores_out == a.scores;
  const int first = wave * R * 64 + lane;  // this thread's slots: first + 64 j
  float score[R];
  int pos[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int i = min(first + 64 * j, a.S_max - 1);
    score[j] = sc[i];
    pos[j] = sp[i];
  }
  const int n = min(max(a.ctx_len[bh / a.Hkv], 0), a.S_max), kept = min(n, a.budget);
  for (int i = t; i < 3 * EV_BINS; i += EV_THREADS) hist[i] = 0;
  if (n <= a.budget) {  // nothing to evict (workgroup-uniform)
    for (int i = t; i < kept; i += EV_THREADS) src[i] = i;
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (!same && first + 64 * j < kept) {
        so[first + 64 * j] = score[j];
        po[first + 64 * j] = pos[j];
      }
    for (int i = kept + t; i < a.S_out; i += EV_THREADS) {
      so[i] = 0.0f;
      po[i] = -1;
    }
    return;
  }
  int newest = INT32_MIN;
#pragma unroll
  for (int j = 0; j < R; ++j)
    if (first + 64 * j < n) newest = max(newest, pos[j]);
  newest = wave_max_int(newest);
  if (lane == 0) red[wave] = newest;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EV_WAVES / 4; ++i) {
    const int4 v = *reinterpret_cast<const int4*>(red + 4 * i);
    newest = max(max(newest, max(v.x, v.y)), max(v.z, v.w));
  }
  uint32_t key[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const bool held = int64_t(pos[j]) > int64_t(newest) - a.recent || pos[j] < a.sink;
    key[j] = held ? 0xffffffffu : ev_rank(score[j]);
  }
  // prefix: the threshold's leading bits; need: its place among the entries that
  // share them
  uint32_t prefix = 0, thr = 0;
  int need = a.budget;
  bool found = false;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    if (found) continue;  // workgroup-uniform
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11, per = (1 << bits) / 64;
    uint32_t* h = hist + pass * EV_BINS;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool in = first + 64 * j < n && (pass == 0 || (key[j] >> (shift + bits)) == prefix);
      const uint64_t m = __ballot(in);
      if (m == 0) continue;
      const int bin = (1 << bits) - 1 - int((key[j] >> shift) & ((1u << bits) - 1));  // from the top
      const int lead = __shfl(bin, __ffsll((unsigned long long)m) - 1, 64);
      uint32_t* p = h + (bin % per) * 64 + bin / per;
      if (__ballot(in && bin == lead) == m) {  // a run of equal scores: one addition
        if (lane == __ffsll((unsigned long long)m) - 1) atomicAdd(p, uint32_t(__popcll(m)));
      } else if (in) {
        atomicAdd(p, 1u);
      }
    }
    __syncthreads();
    if (wave == 0) {  // lane l holds bins [per l, per l + per); first the lane, then the bin
      int sum = 0;
#pragma unroll
      for (int i = 0; i < per; ++i) sum += int(h[i * 64 + lane]);
      const int upto = wave_scan(sum);
      const int at = __ffsll((unsigned long long)__ballot(upto >= need)) - 1;
      const int above = __builtin_amdgcn_readlane(upto - sum, at);
      const int c = lane < per ? int(h[lane * 64 + at]) : 0, incl = above + wave_scan(c);
      const int i = __ffsll((unsigned long long)__ballot(incl >= need)) - 1;
      if (lane == i) {
        sel[pass * 4] = (1 << bits) - 1 - (at * per + i);
        sel[pass * 4 + 1] = incl - c;
        sel[pass * 4 + 2] = c;
      }
    }
    __syncthreads();
    prefix = (prefix << bits) | uint32_t(sel[pass * 4]);
    need -= sel[pass * 4 + 1];
    thr = prefix << shift;
    if (sel[pass * 4 + 2] == need && thr > 0) {  // the whole bin stays
      --thr;
      need = 0;
      found = true;
    }
  }
  // key > thr stays, and of those at thr the first `need` slots
  int eq = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) eq += __popcll(__ballot(first + 64 * j < n && key[j] == thr));
  if (lane == 0) red[EV_WAVES + wave] = eq;
  __syncthreads();
  int all, e = waves_before(red + EV_WAVES, wave, all);
  const uint64_t below = (1ull << lane) - 1;
  uint32_t keep = 0;  // bit j
  int holes = 0, movers = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int i = first + 64 * j;
    const bool at = i < n && key[j] == thr;
    const uint64_t m = __ballot(at);
    const bool k = i < n && (key[j] > thr || (at && e + int(__popcll(m & below)) < need));
    e += __popcll(m);
    keep |= uint32_t(k) << j;
    holes += __popcll(__ballot(!k && i < a.budget));
    movers += __popcll(__ballot(k && i >= a.budget));
  }
  if (lane == 0) {
    red[wave] = holes;  // (the positions there were read two barriers ago)
    red[2 * EV_WAVES + wave] = movers;
  }
  __syncthreads();
  int total, h0 = waves_before(red, wave, total), m0 = waves_before(red + 2 * EV_WAVES, wave, all);
  int rank[R];  // of a hole
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int i = first + 64 * j;
    const bool k = (keep >> j) & 1u, hole = !k && i < a.budget, mover = k && i >= a.budget;
    const uint64_t hm = __ballot(hole), mm = __ballot(mover);
    rank[j] = hole ? h0 + int(__popcll(hm & below)) : -1;
    if (hole) h_slot[rank[j]] = i;
    if (mover) {
      const int r = m0 + int(__popcll(mm & below));
      m_slot[r] = i;
      m_score[r] = score[j];
      m_pos[r] = pos[j];
    }
    h0 += __popcll(hm);
    m0 += __popcll(mm);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int i = first + 64 * j;
    if (i < a.budget) {  // (budget < n: a slot of the cache)
      const int r = rank[j];
      src[i] = r < 0 ? i : m_slot[r];
      if (r >= 0 || !same) {
        so[i] = r < 0 ? score[j] : m_score[r];
        po[i] = r < 0 ? pos[j] : m_pos[r];
      }
    }
  }
  for (int i = a.budget + t; i < a.S_out; i += EV_THREADS) {
    so[i] = 0.0f;
    po[i] = -1;
  }
  if (mvd.k == nullptr) return;
  for (int m = t >> 4; m < total; m += EV_THREADS / 16) {  // 16 lanes a row
    const int64_t base = int64_t(bh) * a.S_max * HD + (t & 15) * 8;
    const int64_t from = base + int64_t(m_slot[m]) * HD, to = base + int64_t(h_slot[m]) * HD;
    const u32x4 kr = ld16(mvd.k + from), vr = ld16(mvd.v + from);
    *reinterpret_cast<u32x4*>(mvd.k + to) = kr;
    *reinterpret_cast<u32x4*>(mvd.v + to) = vr;
  }
}
template <int R>
constexpr int ev_lds() {
  return (3 * EV_BINS + 3 * EV_WAVES + 16 + 4 * R * 512) * 4;
}
static_assert(ev_lds<16>() <= 160 * 1024, "LDS");

// The same for longer caches: the ranks are read again from LDS or memory for
// every pass, the movers' slots go through the workspace.  Bound by one workgroup's
// passes over a (row, kv head), six or more of them (with the moves, into another
// cache, 4 heads: 16,385 entries to 1024 36 us, 16,384 in registers 28; 32,768 to
// 2048 60 us; past EV_LDS_KEYS from memory, 131,072 to 4096 358 us).
__global__ __launch_bounds__(EV_THREADS) void kv_select_long_kernel(const EvArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t ev_smem[];
  uint32_t* hist = ev_smem;                                    // [EV_BINS]
  int* red = reinterpret_cast<int*>(ev_smem + EV_BINS);        // [EV_WAVES]
  int* red2 = red + EV_WAVES;                                  // [EV_WAVES]
  int* sel = red2 + EV_WAVES;                                  // digit, entries above it
  uint32_t* keys = ev_smem + EV_BINS + 2 * EV_WAVES + 16;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int bh = blockIdx.x, b = bh / a.Hkv;
  const int n = min(max(a.ctx_len[b], 0), a.S_max);
  const float* sc = a.scores + int64_t(bh) * a.S_max;
  const int32_t* sp = a.slot_pos + int64_t(bh) * a.S_max;
  float* so = a.scores_out + int64_t(bh) * a.S_out;
  int32_t* po = a.pos_out + int64_t(bh) * a.S_out;
  int32_t* src = a.src + int64_t(bh) * a.budget;
  const bool same = a.scores_out == a.scores;
  const int kept = min(n, a.budget);
  if (n <= a.budget) {  // nothing to evict (workgroup-uniform)
    for (int i = t; i < kept; i += EV_THREADS) {
      src[i] = i;
      if (!same) {
        so[i] = sc[i];
        po[i] = sp[i];
      }
    }
    for (int i = kept + t; i < a.S_out; i += EV_THREADS) {
      so[i] = 0.0f;
      po[i] = -1;
    }
    return;
  }
  int newest = INT32_MIN;
  for (int i = t; i < n; i += EV_THREADS) newest = max(newest, sp[i]);
  for (int d = 1; d < 64; d *= 2) newest = max(newest, __shfl_xor(newest, d, 64));
  if (lane == 0) red[wave] = newest;
  __syncthreads();
  for (int w = 0; w < EV_WAVES; ++w) newest = max(newest, red[w]);
  __syncthreads();
  auto rank_of = [&](int i) {
    const int p = sp[i];
    const bool held = int64_t(p) > int64_t(newest) - a.recent || p < a.sink;
    return held ? 0xffffffffu : ev_rank(sc[i]);
  };
  const bool in_lds = n <= a.lds_keys;
  if (in_lds)
    for (int i = t; i < n; i += EV_THREADS) keys[i] = rank_of(i);
  auto key_of = [&](int i) { return in_lds ? keys[i] : rank_of(i); };
  // radix select: prefix = the threshold's leading bits, need = its place among the
  // entries that share them
  uint32_t prefix = 0;
  int need = a.budget;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    const int bins = 1 << bits;
    for (int i = t; i < bins; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    for (int i = t; i < n; i += EV_THREADS) {
      const uint32_t key = key_of(i);
      if (pass == 0 || (key >> (shift + bits)) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // entries in higher bins than each: thread t owns bins [2 t, 2 t + 2) from the top
    const int b0 = bins - 1 - 2 * t, b1 = b0 - 1;
    const int c0 = b0 >= 0 ? int(hist[b0]) : 0, c1 = b1 >= 0 ? int(hist[b1]) : 0;
    int incl = c0 + c1;
    for (int d = 1; d < 64; d *= 2) {
      const int o = __shfl_up(incl, d, 64);
      if (lane >= d) incl += o;
    }
    if (lane == 63) red[wave] = incl;
    __syncthreads();
    int above = incl - c0 - c1;
    for (int w = 0; w < wave; ++w) above += red[w];
    if (b0 >= 0 && above < need && above + c0 >= need) {
      sel[0] = b0;
      sel[1] = above;
    }
    if (b1 >= 0 && above + c0 < need && above + c0 + c1 >= need) {
      sel[0] = b1;
      sel[1] = above + c0;
    }
    __syncthreads();
    prefix = (prefix << bits) | uint32_t(sel[0]);
    need -= sel[1];
    __syncthreads();
  }
  const uint32_t thr = prefix;  // the first `need` slots at thr stay
  // each wave's run of slots
  const int per = ((n + EV_WAVES - 1) / EV_WAVES + 63) / 64 * 64, w0 = min(n, wave * per), w1 = min(n, w0 + per);
  int eq = 0;
  for (int i0 = w0; i0 < w1; i0 += 64)
    eq += __popcll(__ballot(i0 + lane < w1 && key_of(i0 + lane) == thr));
  if (lane == 0) red[wave] = eq;
  __syncthreads();
  int eq0 = 0;
  for (int w = 0; w < wave; ++w) eq0 += red[w];
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  auto walk = [&](auto&& each) {  // each(slot, kept): every lane of the wave, in slot order
    int e = eq0;
    for (int i0 = w0; i0 < w1; i0 += 64) {
      const int i = i0 + lane;
      const uint32_t key = i < w1 ? key_of(i) : 0u;
      const bool at = i < w1 && key == thr;
      const uint64_t m = __ballot(at);
      const bool keep = i < w1 && (key > thr || (at && e + int(__popcll(m & below)) < need));
      e += __popcll(m);
      each(i, i < w1, keep);
    }
  };
  int holes = 0, movers = 0;
  walk([&](int i, bool in, bool keep) {
    holes += __popcll(__ballot(in && !keep && i < a.budget));
    movers += __popcll(__ballot(in && keep && i >= a.budget));
  });
  if (lane == 0) {
    red[wave] = holes;
    red2[wave] = movers;
  }
  __syncthreads();
  int h0 = 0, m0 = 0;
  for (int w = 0; w < wave; ++w) {
    h0 += red[w];
    m0 += red2[w];
  }
  int32_t* mv = a.movers + int64_t(bh) * a.budget;
  walk([&](int i, bool in, bool keep) {
    const uint64_t hm = __ballot(in && !keep && i < a.budget), mm = __ballot(in && keep && i >= a.budget);
    if (in && i < a.budget) src[i] = keep ? i : -1 - (h0 + int(__popcll(hm & below)));
    if (in && keep && i >= a.budget) mv[m0 + int(__popcll(mm & below))] = i;
    h0 += __popcll(hm);
    m0 += __popcll(mm);
  });
  __syncthreads();
  // the hole of each rank takes the mover of that rank (there are as many)
  for (int i = t; i < a.budget; i += EV_THREADS) {
    int s = src[i];
    if (s < 0) {
      s = mv[-1 - s];
      src[i] = s;
    } else if (same) {
      continue;
    }
    so[i] = sc[s];
    po[i] = sp[s];
  }
  __syncthreads();  // within one cache the tail was read above
  for (int i = a.budget + t; i < a.S_out; i += EV_THREADS) {
    so[i] = 0.0f;
    po[i] = -1;
  }
}

constexpr int EM_SLOTS = 64;  // slots of a workgroup: 16 lanes a row of 256 bytes, 4 rows a lane

struct EmArgs {
  const uint16_t *k, *v;
  uint16_t *k_out, *v_out;
  const int32_t* src;
  const int32_t* ctx_len;
  int Hkv, S_max, S_out, budget;
};

__global__ __launch_bounds__(256) void kv_move_kernel(const EmArgs a) {
  const int bh = blockIdx.y, n = min(max(a.ctx_len[bh / a.Hkv], 0), a.S_max), kept = min(n, a.budget);
  const int c = threadIdx.x & 15, i0 = int(blockIdx.x) * EM_SLOTS + int(threadIdx.x >> 4);
  const bool same = a.k == a.k_out;
  const int32_t* src = a.src + int64_t(bh) * a.budget;
  int from[EM_SLOTS / 16];
#pragma unroll
  for (int j = 0; j < EM_SLOTS / 16; ++j) {
    const int i = i0 + 16 * j;
    const int s = i < kept ? src[i] : -1;
    from[j] = same && s == i ? -1 : s;
  }
  u32x4 kr[EM_SLOTS / 16], vr[EM_SLOTS / 16];
#pragma unroll
  for (int j = 0; j < EM_SLOTS / 16; ++j)
    if (from[j] >= 0) {
      const int64_t at = (int64_t(bh) * a.S_max + from[j]) * HD + c * 8;
      kr[j] = ld16(a.k + at);
      vr[j] = ld16(a.v + at);
    }
#pragma unroll
  for (int j = 0; j < EM_SLOTS / 16; ++j)
    if (from[j] >= 0) {
      const int64_t at = (int64_t(bh) * a.S_out + i0 + 16 * j) * HD + c * 8;
      *reinterpret_cast<u32x4*>(a.k_out + at) = kr[j];
      *reinterpret_cast<u32x4*>(a.v_out + at) = vr[j];
    }
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int qmoe_kv_append(const float* qkv, const qmoe_bf16* q_norm_w, const qmoe_bf16* k_norm_w,
                              const float* rope_cos, const float* rope_sin, int64_t max_pos,
                              const int32_t* positions, const int32_t* slots, int64_t B, int64_t Hq, int64_t Hkv,
                              int64_t D, int64_t S_max, float eps, qmoe_bf16* q_out, qmoe_bf16* k_cache,
                              qmoe_bf16* v_cache, float* scores, int32_t* slot_pos, qmoe_stream_t stream) {
  const char* fn = "qmoe_kv_append";
  QMOE_REQUIRE(q_norm_w && k_norm_w && rope_cos && rope_sin &&
                   (B == 0 || (qkv && positions && slots && q_out && k_cache && v_cache)),
               "%s: null pointer", fn);
  QMOE_REQUIRE(D == HD, "%s: head_dim must be 128 (D=%lld)", fn, (long long)D);
  QMOE_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq < 65536 && Hq + 2 * Hkv < 65536, "%s: bad head counts", fn);
  QMOE_REQUIRE(B >= 0 && B < 65536 && S_max > 0 && S_max < (1ll << 30) && max_pos > 0, "%s: bad B/S_max/max_pos", fn);
  if (B == 0) return QMOE_OK;
  hipLaunchKernelGGL(kv_append_kernel, dim3(unsigned(Hq + 2 * Hkv), unsigned(B)), dim3(64), 0, as_stream(stream),
                     qkv, q_norm_w, k_norm_w, rope_cos, rope_sin, positions, slots, int(Hq), int(Hkv), int(S_max),
                     int(std::min<int64_t>(max_pos, 1ll << 30)), eps, q_out, k_cache, v_cache, scores, slot_pos);
  return hip_status(fn);
}

// Keys of a workgroup: 64, while that makes at most two of them a CU and 64
// records a row (1 x 1100: 10.6 -> 8.3 us), else 256.
static int64_t sd_split(int64_t B, int64_t Hkv, int64_t max_ctx) {
  const int64_t n = (max_ctx + SD_KEYS - 1) / SD_KEYS;
  return n <= 64 && n * B * Hkv <= 512 ? SD_KEYS : SD_KEYS * SD_WAVES;
}
static int64_t sd_bytes(int64_t B, int64_t Hq, int64_t max_ctx, int64_t split) {
  const int64_t n = (max_ctx + split - 1) / split;
  return B * Hq * n * (2 + HD + split) * int64_t(sizeof(float));
}

// (for the split that takes more, so that the size does not hang on Hkv)
extern "C" int64_t qmoe_attn_decode_scored_workspace(int64_t B, int64_t Hq, int64_t D, int64_t max_ctx) {
  if (B < 0 || B >= 65536 || Hq < 0 || Hq >= 65536 * SD_MAX_G || D != HD || max_ctx < 0 || max_ctx >= (1ll << 30))
    return -1;
  if (B * Hq >= (1ll << 31) || B * Hq * max_ctx >= (1ll << 58)) return -1;  // at most 12.2 bytes each, and 1.5 KB a head
  const int64_t few = (max_ctx + SD_KEYS - 1) / SD_KEYS <= 64 && B <= 512 ? sd_bytes(B, Hq, max_ctx, SD_KEYS) : 0;
  return std::max(few, sd_bytes(B, Hq, max_ctx, SD_KEYS * SD_WAVES));
}

extern "C" int qmoe_attn_decode_scored(const qmoe_bf16* q, const qmoe_bf16* k_cache, const qmoe_bf16* v_cache,
                                       const int32_t* ctx_len, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                       int64_t S_max, int64_t max_ctx, float scale, void* workspace,
                                       int64_t workspace_bytes, float* scores, qmoe_bf16* out,
                                       qmoe_stream_t stream) {
  const char* fn = "qmoe_attn_decode_scored";
  QMOE_REQUIRE(B == 0 || (q && k_cache && v_cache && ctx_len && scores && out), "%s: null pointer", fn);
  QMOE_REQUIRE(D == HD, "%s: head_dim must be 128 (D=%lld)", fn, (long long)D);
  QMOE_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= SD_MAX_G && Hkv < 65536,
               "%s: need Hq %% Hkv == 0 and Hq / Hkv <= 16", fn);
  QMOE_REQUIRE(B >= 0 && B < 65536 && S_max > 0 && S_max < (1ll << 30) && B * Hq < (1ll << 31),
               "%s: bad B/S_max", fn);
  QMOE_REQUIRE(max_ctx > 0 && max_ctx <= S_max, "%s: need 0 < max_ctx <= S_max", fn);
  QMOE_REQUIRE(qmoe_attn_decode_scored_workspace(B, Hq, D, max_ctx) >= 0, "%s: B * Hq * max_ctx too large", fn);
  QMOE_REQUIRE(scale > 0.0f && std::isfinite(scale), "%s: scale must be positive and finite", fn);
  if (B == 0) return QMOE_OK;
  const int64_t split = sd_split(B, Hkv, max_ctx), ns = (max_ctx + split - 1) / split;
  const int64_t need = sd_bytes(B, Hq, max_ctx, split);
  QMOE_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %lld bytes, need %lld", fn,
               (long long)workspace_bytes, (long long)need);
  const int64_t n_merge = (B * Hq + 3) / 4, slices = (ns * split + SD_SLICE - 1) / SD_SLICE;
  QMOE_REQUIRE(n_merge + B * Hkv * slices < (1ll << 31), "%s: grid too large", fn);
  QMOE_REQUIRE(aligned16(q, k_cache, v_cache, static_cast<uint8_t*>(workspace), out),
               "%s: operands must be 16-byte aligned", fn);
  const int64_t recs = B * Hq * ns;  // 16-byte pieces first: outputs, logits, then (m, l)
  float* f = static_cast<float*>(workspace);
  SdArgs a{q, k_cache, v_cache, ctx_len, int(B), int(Hq), int(Hkv), int(S_max), int(max_ctx), int(split), int(ns),
           int(ns * split), scale * 1.4426950408889634f, f + recs * (HD + split), f, f + recs * HD, scores, out,
           int(n_merge)};
  const dim3 grid{unsigned(ns), unsigned(Hkv), unsigned(B)};
  if (split == SD_KEYS)
    hipLaunchKernelGGL(attn_scored_kernel<1>, grid, dim3(64), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL(attn_scored_kernel<SD_WAVES>, grid, dim3(SD_WAVES * 64), 0, as_stream(stream), a);
  if (int rc = hip_status(fn)) return rc;
  hipLaunchKernelGGL(attn_scored_finish_kernel, dim3(unsigned(n_merge + B * Hkv * slices)), dim3(256), 0,
                     as_stream(stream), a);
  return hip_status(fn);
}

constexpr int64_t EV_HERE = 256;  // rows that the selection moves itself, at most

template <int R>
static void ev_launch(dim3 grid, const EvArgs& e, const EvMove& mv, hipStream_t s) {
  static const bool attr = [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kv_select_kernel<R>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, ev_lds<R>());
    return true;
  }();
  (void)attr;
  hipLaunchKernelGGL(kv_select_kernel<R>, grid, dim3(EV_THREADS), ev_lds<R>(), s, e, mv);
}

extern "C" int64_t qmoe_kv_evict_workspace(int64_t B, int64_t Hkv, int64_t S_max, int64_t budget) {
  if (B < 0 || B >= 65536 || Hkv < 0 || Hkv >= 65536 || B * Hkv >= 65536 || S_max < 0 || S_max >= (1ll << 30) ||
      budget < 0)
    return -1;
  return 2 * B * Hkv * std::min(budget, S_max) * int64_t(sizeof(int32_t));
}

extern "C" int qmoe_kv_evict(const qmoe_bf16* k_cache, const qmoe_bf16* v_cache, const float* scores,
                             const int32_t* slot_pos, const int32_t* ctx_len, int64_t B, int64_t Hkv, int64_t D,
                             int64_t S_max, int64_t budget, int64_t recent, int64_t sink, void* workspace,
                             int64_t workspace_bytes, int64_t S_out, qmoe_bf16* k_out, qmoe_bf16* v_out,
                             float* scores_out, int32_t* slot_pos_out, qmoe_stream_t stream) {
  const char* fn = "qmoe_kv_evict";
  QMOE_REQUIRE(B == 0 || (k_cache && v_cache && scores && slot_pos && ctx_len && k_out && v_out && scores_out &&
                          slot_pos_out),
               "%s: null pointer", fn);
  QMOE_REQUIRE(D == HD, "%s: head_dim must be 128 (D=%lld)", fn, (long long)D);
  QMOE_REQUIRE(B >= 0 && B < 65536 && Hkv > 0 && Hkv < 65536 && B * Hkv < 65536, "%s: need 0 <= B * Hkv < 65536", fn);
  QMOE_REQUIRE(S_max > 0 && S_max < (1ll << 30) && S_out < (1ll << 30), "%s: bad S_max/S_out", fn);
  QMOE_REQUIRE(budget > 0 && recent >= 0 && sink >= 0 && recent <= budget - sink,
               "%s: need budget > 0 and 0 <= recent + sink <= budget", fn);
  budget = std::min(budget, S_max);
  QMOE_REQUIRE(S_out >= budget, "%s: the destination has %lld slots, the budget is %lld", fn, (long long)S_out,
               (long long)budget);
  const bool same = k_out == k_cache;
  QMOE_REQUIRE(same == (v_out == v_cache) && same == (scores_out == scores) && same == (slot_pos_out == slot_pos) &&
                   (!same || S_out == S_max),
               "%s: the destination is another cache or exactly this one", fn);
  if (B == 0) return QMOE_OK;
  const int64_t need = qmoe_kv_evict_workspace(B, Hkv, S_max, budget);
  QMOE_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %lld bytes, need %lld", fn,
               (long long)workspace_bytes, (long long)need);
  QMOE_REQUIRE(aligned16(k_cache, v_cache, k_out, v_out), "%s: the caches must be 16-byte aligned", fn);
  int32_t* src = static_cast<int32_t*>(workspace);
  const int lds_keys = int(std::min<int64_t>(S_max, EV_LDS_KEYS));
  EvArgs e{scores, slot_pos, ctx_len, int(B), int(Hkv), int(S_max), int(budget),
           int(std::min<int64_t>(recent, 1 << 30)), int(std::min<int64_t>(sink, 1 << 30)), int(S_out), lds_keys,
           scores_out, slot_pos_out, src, src + B * Hkv * budget};
  // in place, with few entries past the budget: 64 rows move at a time
  const bool here = same && S_max <= 16 * EV_THREADS && std::min(budget, S_max - budget) <= EV_HERE;
  const EvMove mv{here ? k_out : nullptr, here ? v_out : nullptr};
  const dim3 grid{unsigned(B * Hkv)};
  if (S_max <= EV_THREADS)
    ev_launch<1>(grid, e, mv, as_stream(stream));
  else if (S_max <= 2 * EV_THREADS)
    ev_launch<2>(grid, e, mv, as_stream(stream));
  else if (S_max <= 4 * EV_THREADS)
    ev_launch<4>(grid, e, mv, as_stream(stream));
  else if (S_max <= 8 * EV_THREADS)
    ev_launch<8>(grid, e, mv, as_stream(stream));
  else if (S_max <= 16 * EV_THREADS)
    ev_launch<16>(grid, e, mv, as_stream(stream));
  else {
    static const bool attr = [] {
      (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kv_select_long_kernel),
                                hipFuncAttributeMaxDynamicSharedMemorySize,
                                (EV_BINS + 2 * EV_WAVES + 16 + EV_LDS_KEYS) * 4);
      return true;
    }();
    (void)attr;
    hipLaunchKernelGGL(kv_select_long_kernel, grid, dim3(EV_THREADS), (EV_BINS + 2 * EV_WAVES + 16 + lds_keys) * 4,
                       as_stream(stream), e);
  }
  if (int rc = hip_status(fn)) return rc;
  if (here) return QMOE_OK;
  EmArgs m{k_cache, v_cache, k_out, v_out, src, ctx_len, int(Hkv), int(S_max), int(S_out), int(budget)};
  hipLaunchKernelGGL(kv_move_kernel, dim3(unsigned((budget + EM_SLOTS - 1) / EM_SLOTS), unsigned(B * Hkv)), dim3(256),
                     0, as_stream(stream), m);
  return hip_status(fn);
}
