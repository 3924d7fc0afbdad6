// Key/value tiles of the attention kernels (head_dim 128): the LDS layout that
// K and V tiles share, the transposing read of V^T fragments, and a flash
// segment, i.e. the loop of one workgroup's 128 query rows over a run of keys.
#pragma once

#include "common.hpp"
#include "mfma_pipe.hpp"

#include <type_traits>

namespace qmoe {

constexpr int HD = 128;  // head_dim

constexpr int AP_KT = 64;                // keys per step
constexpr int AP_ROWB = HD * 2;          // bytes per K / V row in LDS (no pad: chunks are swizzled)
constexpr int AP_TILE = AP_KT * AP_ROWB;  // 16 KB per K or V tile
constexpr float AP_TAU = 8.0f;           // lazy-max slack (log2 units): p < 2^8 between rescales

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// LDS slot of the 16-byte chunk c of K row r.  A fragment read (ds_read_b128)
// takes one chunk of 16 consecutive rows; r % 16 puts them on 16 distinct
// bank groups.
__device__ __forceinline__ int ap_kslot(int r, int c) { return c ^ (r & 15); }
// LDS slot of chunk c of V row r.  A transposing read (ds_read_b64_tr_b16)
// covers, per half-wave, 4 consecutive rows (4-aligned) x 4 consecutive
// chunks (4-aligned), and per 16-lane group 4 rows x 2 chunks; this XOR keeps
// both on distinct bank groups.
__device__ __forceinline__ int ap_vslot(int r, int c) { return c ^ (4 * (r & 3) + 2 * ((r >> 1) & 1)); }

// ds_read_b64_tr_b16: each group of 16 lanes reads a block of 16 x 4 bf16
// (lane j supplies the address of row j: 4 consecutive elements) and lane i
// receives column i % 4 of rows i / 4, i / 4 + 4, i / 4 + 8, i / 4 + 12.
__device__ __forceinline__ s16x4 lds_read_tr16(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}

// Completes this wave's LDS writes before its own lanes read them (a wave's
// DS instructions run in order; this also keeps the compiler from moving
// reads above the writes).
__device__ __forceinline__ void wave_lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// One wave's 32 query rows of a flash loop.  Scores are computed transposed,
// S^T = K . Q^T, so lane l owns query row l % 32 and lanes l, l ^ 32 share it
// (half of a tile's keys each); O^T = V^T . P^T leaves o[db][e] of that row at
// dim 32 db + 8 (e / 4) + 4 (l / 32) + e % 4.
struct FlashRows {
  bf16x8 qf[HD / 16];  // Q^T as the B operand: dims 16 ks + 8 (l / 32) + [0, 8)
  f32x16 o[4];         // unnormalised output
  float m, l;          // running maximum (log2 units) and this lane's share of the row sum

  // qp: this lane's query row, or nullptr for a row past the end (zeros)
  __device__ __forceinline__ void start(const uint16_t* qp, int hl) {
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const u32x4 v = qp ? ld16(qp + ks * 16 + hl * 8) : u32x4{0u, 0u, 0u, 0u};
      qf[ks] = __builtin_bit_cast(bf16x8, v);
    }
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
  }
  // The whole row's sum, in both of its lanes.
  __device__ __forceinline__ float row_sum() const {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
};

constexpr int FL_SMEM = 4 * AP_TILE;  // K0, K1, V0, V1

// Attends a workgroup's 4 x 32 query rows to keys [0, n_keys) of k / v (rows
// of HD bf16; n_keys >= 1), adding to each wave's state.  Lane's row sees keys
// [0, lim]; every row of the wave sees [0, first] and none a key past last
// (wave-uniform; last < 0: the wave has no row, it only helps to load).
//
// K and V tiles of 64 keys go global -> LDS by DMA, two buffers each, rows past
// n_keys as zeros; the S^T MFMAs of step kt + 1 are issued before the softmax
// and the O^T MFMAs of step kt, so that its VALU work runs while the matrix
// pipe is busy; one barrier a step, after which K(kt + 3) and V(kt + 2) are
// requested.  The maximum is lazy: O and l are rescaled only when a row's
// tile maximum exceeds it by more than AP_TAU, so p stays below 2^AP_TAU and
// O / l is the same.  Every wave of the workgroup calls this alike.
//
// The weights are rounded to bf16 for the product with V, whose MFMA takes both
// operands in the cache's type (half a step, 2^-9 to 2^-8 of each weight), and l
// sums them in 32 bits before that.  With the lazy maximum a row's leading weight is
// any value up to 2^8 rather than 1, so it is rounded too: relative error of a
// chunk's outputs against 64 bits 0.0021-0.0023, of which the rounding of the
// output itself is 0.0016-0.0017 (stream_segment, whose maximum is exact: 0.0018).
__device__ __forceinline__ void flash_segment(uint8_t* smem, const uint16_t* k, const uint16_t* v, int n_keys,
                                              int lim, int first, int last, float scale_log2, FlashRows& st) {
  const int t = threadIdx.x, lane = t & 63, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n_kt = (n_keys + AP_KT - 1) / AP_KT;
  const pipe::i32x4 rk = pipe::make_rsrc(k, uint32_t(n_keys) * AP_ROWB);
  const pipe::i32x4 rv = pipe::make_rsrc(v, uint32_t(n_keys) * AP_ROWB);
  // wave w loads rows [16 w, 16 w + 16) of a tile with four instructions of 4
  // rows; lane j fills slot j % 16 of row 16 w + 4 i + j / 16 (the swizzles are
  // their own inverses; from one i to the next the V chunk stays, the K chunk
  // flips bits 2-3)
  const int lr = lane >> 4, ls16 = lane & 15;
  const uint32_t koff = uint32_t((16 * wave + lr) * AP_ROWB + ap_kslot(lr, ls16) * 16);
  const uint32_t voff = uint32_t((16 * wave + lr) * AP_ROWB + ap_vslot(lr, ls16) * 16);
  const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>(smem));
  auto dma_k = [&](int kt, int buf) {
    const uint32_t dst = lds0 + uint32_t(buf * AP_TILE + wave * 4096), adv = uint32_t(kt) * AP_TILE;
#pragma unroll
    for (int i = 0; i < 4; ++i) pipe::dma16(dst + i * 1024, (koff ^ (i * 64)) + (adv + i * 1024), rk, 0);
  };
  auto dma_v = [&](int kt, int buf) {
    const uint32_t dst = lds0 + uint32_t((2 + buf) * AP_TILE + wave * 4096), adv = uint32_t(kt) * AP_TILE;
#pragma unroll
    for (int i = 0; i < 4; ++i) pipe::dma16(dst + i * 1024, voff + (adv + i * 1024), rv, 0);
  };
  auto qk = [&](int buf, f32x16 (&sc)[2]) {
    const uint8_t* kp = smem + buf * AP_TILE + (lane & 31) * AP_ROWB;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const int so = ap_kslot(lane, 2 * ks + hl) * 16;
      const bf16x8 a0 = *reinterpret_cast<const bf16x8*>(kp + so);
      const bf16x8 a1 = *reinterpret_cast<const bf16x8*>(kp + 32 * AP_ROWB + so);
      sc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, st.qf[ks], ks ? sc[0] : f32x16{}, 0, 0, 0);
      sc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a1, st.qf[ks], ks ? sc[1] : f32x16{}, 0, 0, 0);
    }
  };
  // V^T fragments by transposing reads, in the key order of the P^T registers:
  // element jj of lane l is key 16 s + 8 (jj / 4) + 4 (l / 32) + jj % 4
  const int vg = lane >> 4, ve = (lane >> 2) & 3, vq = lane & 3;
  const uint32_t vlane = uint32_t((4 * (vg >> 1) + ve) * AP_ROWB +
                                  (((2 * (vg & 1) + (vq >> 1)) ^ (2 * (ve >> 1))) * 16) + 8 * (vq & 1));
  uint32_t vdb[4];
#pragma unroll
  for (int db = 0; db < 4; ++db) vdb[db] = vlane + uint32_t(64 * (db ^ ve));

  auto softmax_pv = [&](int buf, int kv0, f32x16 (&sc)[2]) {
    const bool live1 = kv0 + 32 <= last;
    if (kv0 + AP_KT - 1 > first) {
      asm volatile("");  // keeps this a branch: the mask is not worth computing on every step
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = kv0 + kb * 32 + (i >> 2) * 8 + hl * 4 + (i & 3);
          if (key > lim) sc[kb][i] = -INFINITY;
        }
    }
    float mx[11];  // maximum as a tree of 3-input maxima
#pragma unroll
    for (int g = 0; g < 11; ++g) {
      const int a = 3 * g, b = 3 * g + 1, c = 3 * g + 2;
      const float va = sc[a >> 4][a & 15], vb = sc[b >> 4][b & 15];
      mx[g] = c < 32 ? fmaxf(fmaxf(va, vb), sc[c >> 4][c & 15]) : fmaxf(va, vb);
    }
    const float m0 = fmaxf(fmaxf(mx[0], mx[1]), mx[2]), m1 = fmaxf(fmaxf(mx[3], mx[4]), mx[5]);
    const float m2 = fmaxf(fmaxf(mx[6], mx[7]), mx[8]), m3 = fmaxf(mx[9], mx[10]);
    float mloc = fmaxf(fmaxf(fmaxf(m0, m1), m2), m3);
    {  // with lane l ^ 32, the other half of the row's keys
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mloc), __float_as_uint(mloc), false, false);
      mloc = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * scale_log2;
    }
    const bool grow = mloc > st.m + AP_TAU;
    if (__builtin_amdgcn_ballot_w64(grow)) {
      const float m_new = grow ? mloc : st.m;
      const float alpha = grow ? __builtin_amdgcn_exp2f(st.m - m_new) : 1.0f;
      st.l *= alpha;
#pragma unroll
      for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) st.o[db][i] *= alpha;
      st.m = m_new;
    }
    const float mb = st.m == -INFINITY ? 0.0f : st.m;  // no key seen yet: every s is -inf
    uint32_t pk[2][8];
    float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[kb][2 * i], scale_log2, -mb));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[kb][2 * i + 1], scale_log2, -mb));
        const bf16x2_t pp = {static_cast<__bf16>(p0), static_cast<__bf16>(p1)};
        pk[kb][i] = __builtin_bit_cast(uint32_t, pp);
        ls[2 * (i & 1)] += p0;
        ls[2 * (i & 1) + 1] += p1;
      }
    st.l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    const uint8_t* vb = smem + (2 + buf) * AP_TILE;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (s >= 2 && !live1) break;
      const u32x4 pw = {pk[s >> 1][(s & 1) * 4], pk[s >> 1][(s & 1) * 4 + 1], pk[s >> 1][(s & 1) * 4 + 2],
                        pk[s >> 1][(s & 1) * 4 + 3]};
      const bf16x8 pb = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const s16x4 v0 = lds_read_tr16(vb + vdb[db] + (16 * s) * AP_ROWB);
        const s16x4 v1 = lds_read_tr16(vb + vdb[db] + (16 * s + 8) * AP_ROWB);
        const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        st.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb, st.o[db], 0, 0, 0);
      }
    }
  };

  __syncthreads();  // an earlier segment's LDS reads are done
  dma_k(0, 0);
  dma_v(0, 0);
  if (n_kt > 1) {
    dma_k(1, 1);
    dma_v(1, 1);
    pipe::wait_vm<4>();
  } else {
    pipe::wait_vm<0>();
  }
  __syncthreads();  // K(0), V(0), K(1) visible
  // end of step kt: K(kt + 2) and V(kt + 1) have landed; K(kt + 1)'s and V(kt)'s
  // buffers are free
  auto turn = [&](int kt) {
    const int buf = kt & 1;
    pipe::wait_vm<0>();
    __syncthreads();
    if (kt + 3 < n_kt) dma_k(kt + 3, buf ^ 1);
    if (kt + 2 < n_kt) dma_v(kt + 2, buf);
  };
  f32x16 sc[2], sn[2];
  qk(0, sc);
  if (n_kt > 2) {
    __syncthreads();  // every wave is done with K(0)'s buffer
    dma_k(2, 0);
  }
  // steps in pairs, the score registers swapping roles
  auto one = [&](int kt, f32x16 (&cur)[2], f32x16 (&nxt)[2], auto has_next) {
    const int kv0 = kt * AP_KT, buf = kt & 1;
    if constexpr (decltype(has_next)::value) qk(buf ^ 1, nxt);
    if (kv0 <= last) softmax_pv(buf, kv0, cur);
    turn(kt);
  };
  int kt = 0;
  for (; kt + 2 < n_kt; kt += 2) {
    one(kt, sc, sn, std::true_type{});
    one(kt + 1, sn, sc, std::true_type{});
  }
  if (kt + 1 < n_kt) {
    one(kt, sc, sn, std::true_type{});
    one(kt + 1, sn, sc, std::false_type{});
  } else {
    one(kt, sc, sn, std::false_type{});
  }
}

// Few query rows (up to 32) over many keys, where the keys' stream is what costs:
// every wave of the workgroup holds the same rows and takes its own 64-key tiles
// w, w + 4, ... of keys [0, n_keys) of k / v.  K rows go from memory straight
// into A-operand registers and V by DMA into the wave's own LDS tile, every load
// of a tile in flight at once and no barrier between the waves; flash_join adds
// up their states.  Lane's row sees keys [0, lim].  Weights in bf16 for the MFMA with V
// and l in 32 bits, as in flash_segment.
__device__ __forceinline__ void stream_segment(uint8_t* smem, const uint16_t* k, const uint16_t* v, int n_keys,
                                               int lim, float scale_log2, FlashRows& st) {
  const int lane = threadIdx.x & 63, col = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  uint8_t* vb = smem + wave * AP_TILE;
  const int vg = lane >> 4, ve = (lane >> 2) & 3, vq = lane & 3;
  const uint32_t vlane = uint32_t((4 * (vg >> 1) + ve) * AP_ROWB +
                                  (((2 * (vg & 1) + (vq >> 1)) ^ (2 * (ve >> 1))) * 16) + 8 * (vq & 1));
  const pipe::i32x4 rv = pipe::make_rsrc(v, uint32_t(n_keys) * AP_ROWB);  // rows past the end read as zeros
  const uint32_t lds = uint32_t(reinterpret_cast<uintptr_t>(smem)) + uint32_t(wave * AP_TILE);
  const uint32_t voff = uint32_t((lane >> 4) * AP_ROWB + ap_vslot(lane >> 4, lane & 15) * 16);
#pragma unroll 1
  for (int k0 = wave * AP_KT; k0 < n_keys; k0 += 4 * AP_KT) {
    const int last = min(AP_KT, n_keys - k0) - 1;  // rows past it repeat it (their p is 0)
    u32x4 ka[2][HD / 16];
    wave_lds_sync();  // the last tile's V reads are done
#pragma unroll
    for (int i = 0; i < 16; ++i) pipe::dma16(lds + i * 1024, voff + uint32_t(k0 + 4 * i) * AP_ROWB, rv, 0);
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      const uint16_t* kp = k + int64_t(k0 + min(mb * 32 + col, last)) * HD + hl * 8;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) ka[mb][ks] = ld16(kp + ks * 16);
    }
    f32x16 sc[2];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb) {
      sc[mb] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        sc[mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, ka[mb][ks]), st.qf[ks], sc[mb], 0,
                                                         0, 0);
    }
    const int see = min(lim - k0, last);
    float m = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int key = mb * 32 + (e >> 2) * 8 + hl * 4 + (e & 3);
        sc[mb][e] = key <= see ? sc[mb][e] * scale_log2 : -INFINITY;
        m = fmaxf(m, sc[mb][e]);
      }
    {
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
      m = fmaxf(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])), st.m);
    }
    const float mz = m == -INFINITY ? 0.0f : m;  // no key seen yet
    const float alpha = __builtin_amdgcn_exp2f(st.m - mz);
    st.m = m;
    st.l *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) st.o[db][i] *= alpha;
    uint32_t pk[2][8];
    float l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(sc[mb][2 * i] - mz);
        const float p1 = __builtin_amdgcn_exp2f(sc[mb][2 * i + 1] - mz);
        l0 += p0;
        l1 += p1;
        const bf16x2_t pp = {static_cast<__bf16>(p0), static_cast<__bf16>(p1)};
        pk[mb][i] = __builtin_bit_cast(uint32_t, pp);
      }
    st.l += l0 + l1;
    pipe::wait_vm<0>();  // V in LDS
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
        const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        st.o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, pb, st.o[db], 0, 0, 0);
      }
    }
  }
}

// The four waves' states of the same rows into wave 0's, through LDS in register
// order (18 values of 64 lanes a chunk of 4): waves 2 and 3 into 0 and 1, then
// wave 1 into 0.
__device__ __forceinline__ void flash_join(uint8_t* smem, FlashRows& st) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int REC = 64 * (4 * 16 + 2);  // floats of a state
  static_assert(2 * REC * 4 <= FL_SMEM, "two states fit");
  auto put = [&](float* p) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(p + ((db * 4 + g) * 64 + lane) * 4) =
            make_float4(st.o[db][g * 4], st.o[db][g * 4 + 1], st.o[db][g * 4 + 2], st.o[db][g * 4 + 3]);
    *reinterpret_cast<float2*>(p + 64 * 64 + lane * 2) = make_float2(st.m, st.l);
  };
  auto take = [&](const float* p) {
    const float2 ml = *reinterpret_cast<const float2*>(p + 64 * 64 + lane * 2);
    const float m = fmaxf(st.m, ml.x), mz = m == -INFINITY ? 0.0f : m;
    const float a = __builtin_amdgcn_exp2f(st.m - mz), b = __builtin_amdgcn_exp2f(ml.x - mz);
    st.m = m;
    st.l = st.l * a + ml.y * b;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 o = *reinterpret_cast<const float4*>(p + ((db * 4 + g) * 64 + lane) * 4);
        st.o[db][g * 4] = fmaf(st.o[db][g * 4], a, o.x * b);
        st.o[db][g * 4 + 1] = fmaf(st.o[db][g * 4 + 1], a, o.y * b);
        st.o[db][g * 4 + 2] = fmaf(st.o[db][g * 4 + 2], a, o.z * b);
        st.o[db][g * 4 + 3] = fmaf(st.o[db][g * 4 + 3], a, o.w * b);
      }
  };
  float* buf = reinterpret_cast<float*>(smem);
  __syncthreads();  // the V tiles are free
  if (wave >= 2) put(buf + (wave - 2) * REC);
  __syncthreads();
  if (wave < 2) take(buf + wave * REC);
  __syncthreads();
  if (wave == 1) put(buf);
  __syncthreads();
  if (wave == 0) take(buf);
}

}  // namespace qmoe
