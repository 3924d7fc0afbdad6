// Attention with a window, over a cache in bf16 or in 4 bits (head_dim 128): few query
// rows over many keys, where the cache's stream is what costs.  Many rows go to the
// tiles of attn_rows.hip.
//
// A wave takes 64 keys at a time and up to 16 packed query rows (query-major, then
// the G = Hq / Hkv heads of the group), on v_mfma_f32_16x16x32_bf16:
//   S^T [keys x rows] = K . Q^T     O^T [dims x rows] += V^T . P^T
// Numbers of 4 bits become bf16 in registers (v_cvt_scalef32_pk_bf16_fp4, two a step
// with their power; exact), so queries and products are those of a bf16 cache.
//
// Work: 4 * 128 flops a (query head, key), 512 bytes a (kv head, key) in bf16 and 136 in 4
// bits.  8 query heads on a kv head are 8 flops a byte, or 30: the stream from memory
// bounds a long batch in bf16 (32 rows that see 4100 keys each, 269 MB in 49 us and 5 for
// the merge, 5.0 TB/s in all, of a large copy's 5.2) and a very long one in 4 bits (64 rows
// of up to 32768, 714 MB in 138 us, 5.2 TB/s).  Shorter ones in 4 bits are that rate and 11 us of
// launches, first loads, joins and the merge (32 rows of up to 8192 25 us, of up to 16384
// 42).  Few keys are a chain: lengths, queries and keys, one step or two (of 3300 cycles in 4
// bits: 128 conversions, 32 products, 16 exponentials, V through LDS), the join (one row of
// 800 in 4 bits 9 us), and in it what one CU takes in, 19-24 bytes a cycle, for which a row's
// keys in bf16 go to many CUs (516 keys, 4 heads: 9 waves each by itself 7.7 us, 3 workgroups
// of 4 waves 9.9, in a graph).
#include "attn_tile.hpp"
#include "common.hpp"
#include "kv4.hpp"
#include "window.hpp"

#include <type_traits>

namespace qmoe {

constexpr int AS_ROWS = 16;             // query rows of an item
constexpr int AS_TILE = 64;             // keys of a wave's step
constexpr int AS_REC = 2 * AS_ROWS + AS_ROWS * HD;  // record of a piece: (m, l) of the rows, O in register order
constexpr int AS_CUT = 4;               // waves of a workgroup that takes a share of the keys

struct AsArgs {
  const uint16_t *q, *k, *v;
  Cache4 c;  // instead of k and v
  WinArgs win;
  int B, Hq, Hkv, G, rts;  // G: Hq / Hkv; rts: row tiles of a (sequence, kv head)
  int waves, runs, run;  // waves of a workgroup; runs of `run` keys that an item is cut into
  int wgs;               // or workgroups that share all items' keys evenly (0: runs)
  uint32_t g_magic;
  float scale_log2;
  float* part;  // [runs][rts][B][Hkv][AS_REC], when runs > 1, or [wgs][2][AS_REC]
  uint16_t* out;
};

// The keys that an item's queries see, from its first row r0 to its last, r1.  In a
// cache of 4 bits the gap begins at a multiple of 4, so that four keys from a
// multiple of 4 on are rows in a row; the run's rows [stay, hid) are then some that
// no query sees.
struct AsRun {
  WinRow first, last;
  Gap gap;
  int stay, hid, n;
};
template <bool FOUR>
__device__ __forceinline__ AsRun as_run(const AsArgs& a, int b, int r0, int r1) {
  AsRun k;
  k.first = win_row(a.win, b, ar_div(r0, a.g_magic));
  k.last = win_row(a.win, b, ar_div(r1, a.g_magic));
  k.stay = min(a.win.sink, k.last.end);
  const int at = FOUR ? (k.stay + 3) & ~3 : k.stay;
  k.gap = Gap{at, max(k.first.low - at, 0)};
  k.n = k.first.low <= at ? k.last.end : at + max(k.last.end - k.first.low, 0);
  k.hid = k.first.low <= at ? max(k.first.low, k.stay) : at;
  return k;
}

// The work in steps of AS_CUT waves' tiles, items (row tile fastest, then kv head, then
// sequence) one after another; an item has one step at least.  Every workgroup takes
// an equal share of all of them, so that lengths of any kind fill the GPU evenly:
// workgroup w of W the steps [w T / W, (w + 1) T / W).  For caches of 4 bits (a share's
// places in the cache beside bf16's tiles are more than the registers hold).
constexpr int AS_STEP = AS_CUT * AS_TILE;
__device__ __forceinline__ int as_steps(const AsArgs& a, int b, int rt) {
  const int r0 = rt * AS_ROWS, rows = a.win.S * a.G;
  const int n = as_run<true>(a, b, r0, min(r0 + AS_ROWS, rows) - 1).n;
  return max((n + AS_STEP - 1) / AS_STEP, 1);
}
__device__ __forceinline__ int as_row_steps(const AsArgs& a, int b) {  // of one kv head
  int n = 0;
  for (int rt = 0; rt < a.rts; ++rt) n += as_steps(a, b, rt);
  return n;
}
struct AsTotal {
  int T, W;
  __device__ __forceinline__ int begin(int w) const { return int(int64_t(w) * T / W); }
  __device__ __forceinline__ int owner(int step) const { return int((int64_t(step + 1) * W - 1) / T); }
};
__device__ __forceinline__ int wave_scan(int v) {  // inclusive
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(1), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(2), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(4), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_SHR(8), 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_BCAST15, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, QMOE_DPP_ROW_BCAST31, 0xc, 0xf, false);
  return v;
}
// Sums the steps of all sequences, and finds the place that `find` says yes to, given
// the total, a sequence, its first step and its number of steps.  Every wave does it
// for itself, 64 sequences at a time.
struct AsPlace {
  int b, first;
};
template <class Find>
__device__ __forceinline__ AsTotal as_total(const AsArgs& a, AsPlace* place, Find find) {
  const int lane = threadIdx.x & 63;
  AsTotal tot{0, 0};
  int n = 0, upto = 0;
  for (int c = 0; c < a.B; c += 64) {
    n = c + lane < a.B ? as_row_steps(a, c + lane) * a.Hkv : 0;
    upto = wave_scan(n);
    tot.T += __builtin_amdgcn_readlane(upto, 63);
  }
  tot.W = min(a.wgs, tot.T);
  int before = 0;
  *place = AsPlace{0, 0};
  for (int c = 0; c < a.B; c += 64) {
    if (a.B > 64) {
      n = c + lane < a.B ? as_row_steps(a, c + lane) * a.Hkv : 0;
      upto = wave_scan(n);
    }
    const int first = before + upto - n;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(c + lane < a.B && find(tot, c + lane, first, n));
    if (hit) {
      const int l = __builtin_ctzll(hit);
      *place = AsPlace{c + l, __builtin_amdgcn_readlane(first, l)};
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return tot;
}

// A wave's 64 keys on their way: loads of the next tile's K go out once this one's
// products are issued, its V's once this one's is in LDS.  rows: rows of the cache
// that may be read; past them everything is zero.
// 4 bits: lane (r = lane % 16, g = lane / 16) holds block g of the keys 4 r + [0, 4),
// whose powers are 16 bytes in a row.
struct AsTile4 {
  __amdgpu_buffer_rsrc_t rk, rv, rks, rvs;
  u32x4 k[4], ks, v[4], vs;
  Gap gap;
  int stay, hid;
  __device__ __forceinline__ void start(const AsArgs& a, const AsRun& run, int64_t base, int rows) {
    rk = kv4_rsrc(a.c.k + base * KV4_ROWB, int64_t(rows) * KV4_ROWB);
    rv = kv4_rsrc(a.c.v + base * KV4_ROWB, int64_t(rows) * KV4_ROWB);
    rks = kv4_rsrc(a.c.ks + base * 4, int64_t(rows) * 4);
    rvs = kv4_rsrc(a.c.vs + base * 4, int64_t(rows) * 4);
    gap = run.gap;
    stay = run.stay;
    hid = run.hid;
  }
  __device__ __forceinline__ void load_k(int t0, int r, int g) {
    const uint32_t rr = uint32_t(gap.row(t0 + 4 * r));
#pragma unroll
    for (int j = 0; j < 4; ++j) k[j] = kv4_ld16(rk, (rr + j) * KV4_ROWB + g * 16);
    ks = kv4_ld16(rks, rr * 4);
  }
  __device__ __forceinline__ void load_v(int t0, int r, int g) {
    const uint32_t rr = uint32_t(gap.row(t0 + 4 * r));
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = kv4_ld16(rv, (rr + j) * KV4_ROWB + g * 16);
    vs = kv4_ld16(rvs, rr * 4);
  }
  // K of the keys 4 r + j as A operands: step ks holds dims dim(g, ks) + [0, 8)
  static __device__ __forceinline__ int dim(int g, int ks) { return 32 * g + 8 * ks; }
  __device__ __forceinline__ void keys(int j, int g, u32x4 (&c)[4]) const {
    kv4_chunks(k[j], kv4_scale((ks[j] >> (8 * g)) & 255u), c);
  }
  // V to LDS
  __device__ __forceinline__ void put_v(uint8_t* vt, int t0, int r, int g) const {
    // chunk pair 2 g + i of key 4 r + j is in place at[i ^ j]
    uint32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      at[i] = uint32_t(r * 4 * AP_ROWB + (((2 * g) ^ ((r & 3) | ((r >> 2) & 1) << 2)) ^ i) * 32);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t p = (vs[j] >> (8 * g)) & 255u;
      if (t0 < hid && t0 + AS_TILE > stay) {  // rows that no query sees add 0, whatever they hold
        const int rw = gap.row(t0 + 4 * r + j);
        p = rw >= stay && rw < hid ? 0u : p;
      }
      u32x4 c[4];
      kv4_chunks(v[j], kv4_scale(p), c);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<u32x4*>(vt + at[(i >> 1) ^ j] + j * AP_ROWB + (i & 1) * 16) = c[i];
    }
  }
};
// bf16: K as A operands straight from memory, 64 bytes of 16 rows an instruction; V as
// whole rows, four an instruction.
struct AsTile16 {
  __amdgpu_buffer_rsrc_t rk, rv;
  u32x4 k[4][4], v[16];
  Gap gap;
  __device__ __forceinline__ void start(const AsArgs& a, const AsRun& run, int64_t base, int rows) {
    rk = kv4_rsrc(reinterpret_cast<const uint8_t*>(a.k + base * HD), int64_t(rows) * AP_ROWB);
    rv = kv4_rsrc(reinterpret_cast<const uint8_t*>(a.v + base * HD), int64_t(rows) * AP_ROWB);
    gap = run.gap;
  }
  __device__ __forceinline__ void load_k(int t0, int r, int g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t at = uint32_t(gap.row(t0 + 4 * r + j)) * AP_ROWB + g * 16;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) k[j][ks] = kv4_ld16(rk, at + ks * 64);
    }
  }
  __device__ __forceinline__ void load_v(int t0, int r, int g) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = kv4_ld16(rv, uint32_t(gap.row(t0 + 4 * i + g)) * AP_ROWB + r * 16);
  }
  static __device__ __forceinline__ int dim(int g, int ks) { return 32 * ks + 8 * g; }
  __device__ __forceinline__ void keys(int j, int g, u32x4 (&c)[4]) const {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) c[ks] = k[j][ks];
  }
  __device__ __forceinline__ void put_v(uint8_t* vt, int t0, int r, int g) const {
    // chunk r of row 4 i + g: its pair's place goes with g ^ i % 4 and i / 4 % 2
    const uint32_t at = uint32_t(g * AP_ROWB + ((r * 16) ^ (g * 32)));
#pragma unroll
    for (int i = 0; i < 16; ++i)
      *reinterpret_cast<u32x4*>(vt + (at ^ ((i & 3) * 32 + ((i >> 2) & 1) * 128)) + i * 4 * AP_ROWB) = v[i];
  }
};

// V passes through LDS in bf16, row = key, 256 bytes; the pair p of 16-byte chunks sits
// at p ^ (((key ^ key / 4) % 4) + 4 (key / 16 % 2)), so that 8 lanes' writes (keys
// 4 r + j of 8 consecutive r, or 8 chunks of a key) and a half-wave's transposing reads
// (keys 16 g + [0, 4) of two g) fall into eight different places.
//
// A piece: the keys [k0, k1) of the item (b, kvh, rt), as output, or where they are not
// all of the item's as the record `part`.
template <bool FOUR, int WAVES>
__device__ __forceinline__ void as_piece(const AsArgs& a, const AsRun& kr, int b, int kvh, int rt, int k0, int k1,
                                         float* part, uint8_t (*smem)[AS_TILE * AP_ROWB], float2 (*sml)[AS_ROWS]) {
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int r0 = rt * AS_ROWS, r1 = min(r0 + AS_ROWS, a.win.S * a.G) - 1;
  const Gap gap = kr.gap;
  const int row = min(r0 + r, r1), sq = ar_div(row, a.g_magic);
  const bool live = r0 + r <= r1;
  const int64_t qrow = (int64_t(b) * a.win.S + sq) * a.Hq + kvh * a.G + (row - sq * a.G);
  using Tile = std::conditional_t<FOUR, AsTile4, AsTile16>;
  // Q^T as B operands, in the order of the K operands' dims (ahead of the cache's loads,
  // behind which the first product would wait for it)
  bf16x8 qf[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const u32x4 w = live ? ld16(a.q + qrow * HD + Tile::dim(g, ks)) : u32x4{0u, 0u, 0u, 0u};
    qf[ks] = __builtin_bit_cast(bf16x8, w);
  }
  __builtin_amdgcn_sched_barrier(0);
  // this lane's row sees the keys [0, stay) and [all, ...) up to row own.end
  const WinRow own = win_row(a.win, b, sq);
  const int all = own.low <= a.win.sink ? 0 : gap.key(own.low);
  // every row of the item sees the keys [from, upto)
  const int from = kr.last.low <= a.win.sink ? 0 : gap.key(kr.last.low);
  const int upto = min(gap.key(kr.first.end - 1) + 1, k1);

  Tile tile;
  const int w0 = k0 + wave * AS_TILE;
  if (k0 < k1)
    tile.start(a, kr, (int64_t(b) * a.Hkv + kvh) * a.win.S_max, min(gap.row(k1 - 1) + 1, a.win.S_max));
  if (w0 < k1) {
    tile.load_k(w0, r, g);
    tile.load_v(w0, r, g);
  }
  f32x4 o[8];  // O^T: dims 16 dt + 4 g + [0, 4) of row r
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;
  uint8_t* vt = smem[wave];
  // transposing reads: 16-lane group g takes keys 16 g + 8 m + 4 h + [0, 4), dims
  // 16 dt + [0, 16), from place rat[dt ^ (2 m + h)]
  const int jr = (lane >> 2) & 3;
  uint32_t rat[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    rat[i] = uint32_t((16 * g + jr) * AP_ROWB + (i ^ (jr | (g & 1) << 2)) * 32 + (lane & 3) * 8);

#pragma unroll 1
  for (int t0 = w0; t0 < k1; t0 += WAVES * AS_TILE) {
    const int t1 = t0 + WAVES * AS_TILE;
    f32x4 sc[4];  // S^T: keys 16 g + 4 i + j of row r
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u32x4 c[4];
      tile.keys(j, g, c);
      sc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
        sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c[ks]), qf[ks], sc[j], 0, 0, 0);
    }
    if (t1 < k1) tile.load_k(t1, r, g);
    wave_lds_sync();  // the last tile's V reads are done
    tile.put_v(vt, t0, r, g);
    if (t1 < k1) tile.load_v(t1, r, g);
    if (t0 < from || t0 + AS_TILE > upto) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = t0 + 16 * g + 4 * i + j;
          const bool see = key < k1 && gap.row(key) < own.end && (key >= all || key < kr.stay);
          sc[j][i] = see ? sc[j][i] : -INFINITY;
        }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fmaxf(fmaxf(sc[j][0], sc[j][1]), fmaxf(sc[j][2], sc[j][3])));
    mx *= a.scale_log2;
    if (__builtin_amdgcn_ballot_w64(mx > m + AP_TAU)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float to = fmaxf(m, mx), alpha = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      m = to;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[dt][i] *= alpha;
    }
    const float mz = m == -INFINITY ? 0.0f : m;
    float ls[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t pw[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[2 * jj][i], a.scale_log2, -mz));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[2 * jj + 1][i], a.scale_log2, -mz));
        ls[2 * jj] += p0;
        ls[2 * jj + 1] += p1;
        const bf16x2_t pp = {static_cast<__bf16>(p0), static_cast<__bf16>(p1)};
        pw[i >> 1][(i & 1) * 2 + jj] = __builtin_bit_cast(uint32_t, pp);
      }
    l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    wave_lds_sync();  // V in LDS
#pragma unroll
    for (int mm = 0; mm < 2; ++mm) {
      const u32x4 pq = {pw[mm][0], pw[mm][1], pw[mm][2], pw[mm][3]};
      const bf16x8 pb = __builtin_bit_cast(bf16x8, pq);
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const s16x4 v0 = lds_read_tr16(vt + rat[dt ^ (2 * mm)] + (8 * mm) * AP_ROWB);
        const s16x4 v1 = lds_read_tr16(vt + rat[dt ^ (2 * mm + 1)] + (8 * mm + 4) * AP_ROWB);
        const bf16x8 va = __builtin_bit_cast(bf16x8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
        o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pb, o[dt], 0, 0, 0);
      }
    }
  }

  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if constexpr (WAVES == 1) {  // nothing to join
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    if (!live) return;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      if (part)
        *reinterpret_cast<f32x4*>(part + 2 * AS_ROWS + (dt * 64 + lane) * 4) = o[dt];
      else
        *reinterpret_cast<u32x2*>(a.out + qrow * HD + dt * 16 + g * 4) =
            u32x2{pack_bf16x2(o[dt][0] * inv, o[dt][1] * inv), pack_bf16x2(o[dt][2] * inv, o[dt][3] * inv)};
    }
    if (part && g == 0) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(m, l);
    return;
  }
  // the waves' states of the same rows: each wave joins its share of the eight dim tiles
  __syncthreads();  // V tiles free
  float* rec = reinterpret_cast<float*>(&smem[0][0]);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(rec + ((wave * 8 + dt) * 64 + lane) * 4) = o[dt];
  if (g == 0) sml[wave][r] = make_float2(m, l);
  __syncthreads();
  float M = -INFINITY, L = 0.0f, wt[WAVES];
#pragma unroll
  for (int w = 0; w < WAVES; ++w) M = fmaxf(M, sml[w][r].x);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const float2 ml = sml[w][r];
    wt[w] = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
    L = fmaf(wt[w], ml.y, L);
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
  for (int i = 0; i < 8 / WAVES; ++i) {
    const int dt = wave * (8 / WAVES) + i;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(rec + ((w * 8 + dt) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(wt[w], v[e], sum[e]);
    }
    if (!live) continue;
    if (part)
      *reinterpret_cast<f32x4*>(part + 2 * AS_ROWS + (dt * 64 + lane) * 4) = sum;
    else
      *reinterpret_cast<u32x2*>(a.out + qrow * HD + dt * 16 + g * 4) =
          u32x2{pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv)};
  }
  if (part && wave == 0 && g == 0) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(M, L);
}

// 64 keys a step: 16 loads of 16 bytes a lane in flight for the next K and V in bf16 (the
// 243 registers are what two waves a SIMD have) and 10 in 4 bits.  16 query rows, since a
// group has 8 heads: of 32 x 32 products three quarters would be of rows that are none.
// Tried for 4 bits and not kept: the next tile but one in flight too (32 x 8192 27 -> 29 us,
// 1 x 800 9.2 -> 10.1); V converted behind the first products (the same time); keys in
// 4 bits and queries as two terms in 8 for the scaled products (their sums are aligned
// to the largest term: errors of 8e-5 of the terms' magnitudes).
//
// Workgroup = (kv head, sequence, run of a row tile): heads and sequences are fastest, so
// the row tiles that share a head's keys are on one XCD when there are a multiple of 8
// of those.
template <bool FOUR, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == 8 ? 1 : 2) void attn_stream_kernel(const AsArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[WAVES][AS_TILE * AP_ROWB];
  __shared__ float2 sml[WAVES][AS_ROWS];
  const int kvh = blockIdx.x, b = blockIdx.y, z = blockIdx.z;
  const int run = a.rts == 1 ? z : z / a.rts, rt = z - run * a.rts;
  const int r0 = rt * AS_ROWS, r1 = min(r0 + AS_ROWS, a.win.S * a.G) - 1;
  const AsRun kr = as_run<FOUR>(a, b, r0, r1);
  const int k0 = run * a.run;
  if (run > 0 && k0 >= kr.n) return;  // the merge knows how many runs there are
  float* part = a.runs > 1 ? a.part + ((int64_t(z) * a.B + b) * a.Hkv + kvh) * AS_REC : nullptr;
  as_piece<FOUR, WAVES>(a, kr, b, kvh, rt, k0, min(kr.n, k0 + a.run), part, smem, sml);
}

// Workgroup = its share of all steps: the end of an item, whole items, the beginning of
// another.  (64 x 32768: 126-141 us; with runs of equal numbers of steps an item 150.)
__global__ __launch_bounds__(AS_CUT * 64, 8 / AS_CUT) void attn_stream_cut_kernel(const AsArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[AS_CUT][AS_TILE * AP_ROWB];
  __shared__ float2 sml[AS_CUT][AS_ROWS];
  const int w = int(blockIdx.x);
  AsPlace at;
  const AsTotal tot = as_total(a, &at, [&](const AsTotal& t, int, int first, int n) {
    const int s = w < t.W ? t.begin(w) : -1;
    return s >= first && s < first + n;
  });
  if (w >= tot.W) return;
  int s = tot.begin(w);
  const int end = tot.begin(w + 1);
  int b = at.b, kvh = 0, rt = 0, off = s - at.first;  // steps of the sequence before s
  {
    const int per = as_row_steps(a, b);
    kvh = off / per;
    off -= kvh * per;
    for (int n; off >= (n = as_steps(a, b, rt)); ++rt) off -= n;
  }
  while (s < end) {
    const int r0 = rt * AS_ROWS, r1 = min(r0 + AS_ROWS, a.win.S * a.G) - 1;
    const AsRun kr = as_run<true>(a, b, r0, r1);
    const int steps = max((kr.n + AS_STEP - 1) / AS_STEP, 1), take = min(steps - off, end - s);
    float* part = take == steps ? nullptr : a.part + (int64_t(w) * 2 + (off == 0)) * AS_REC;
    as_piece<true, AS_CUT>(a, kr, b, kvh, rt, off * AS_STEP, min(kr.n, (off + take) * AS_STEP), part, smem, sml);
    s += take;
    off = 0;
    if (++rt == a.rts) {
      rt = 0;
      if (++kvh == a.Hkv) {
        kvh = 0;
        ++b;
      }
    }
    __syncthreads();  // LDS free for the next piece
  }
}

// Joins the pieces of an item's rows: workgroup = (item, dim tile); wave v takes the
// pieces v, v + 4, ..., four at a time.  Bound by latency: one round trip for the lengths
// and one for the records (3 items 2.3 us, 32 x 4 items of 4 pieces 3.9, of shares 6.6).
template <bool FOUR, bool CUT>
__global__ __launch_bounds__(256) void attn_stream_merge_kernel(const AsArgs a) {
  __shared__ f32x4 so[4][64];
  __shared__ float2 sml[4][64];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
  const int dt = int(blockIdx.x) & 7, kvh = int(blockIdx.x) >> 3, b = blockIdx.y, rt = blockIdx.z;
  const int rows = a.win.S * a.G, r0 = rt * AS_ROWS;
  int pieces;
  const float *p0, *p1;  // the first piece's record and the second one's, then every `next`
  int64_t next;
  if constexpr (CUT) {
    AsPlace at;
    const AsTotal tot = as_total(a, &at, [&](const AsTotal&, int c, int, int) { return c == b; });
    int first = at.first + kvh * as_row_steps(a, b);
    for (int i = 0; i < rt; ++i) first += as_steps(a, b, i);
    // workgroup w0 began the item (its second record), the next ones went on (their first)
    const int w0 = tot.owner(first);
    pieces = tot.owner(first + as_steps(a, b, rt) - 1) - w0 + 1;
    if (pieces == 1) return;  // whole, and already output
    next = 2 * AS_REC;
    p0 = a.part + (int64_t(w0) * 2 + 1) * AS_REC;
    p1 = p0 + AS_REC;
  } else {
    pieces = max((as_run<FOUR>(a, b, r0, min(r0 + AS_ROWS, rows) - 1).n + a.run - 1) / a.run, 1);
    next = int64_t(a.B) * a.Hkv * a.rts * AS_REC;
    p0 = a.part + ((int64_t(rt) * a.B + b) * a.Hkv + kvh) * AS_REC;
    p1 = p0 + next;
  }
  const int row = r0 + r;
  float M = -INFINITY, L = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < rows) {
    for (int i0 = wave; i0 < pieces; i0 += 16) {
      float2 ml[4];
      f32x4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 4 * u, j = min(i, pieces - 1);
        const float* q = j == 0 ? p0 : p1 + (j - 1) * next;
        ml[u] = *reinterpret_cast<const float2*>(q + 2 * r);
        v[u] = *reinterpret_cast<const f32x4*>(q + 2 * AS_ROWS + (dt * 64 + lane) * 4);
        if (i >= pieces) ml[u] = make_float2(-INFINITY, 0.0f);
      }
      const float to = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M);
      const float mz = to == -INFINITY ? 0.0f : to, al = __builtin_amdgcn_exp2f(M - mz);
      M = to;
      L *= al;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= al;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float wt = __builtin_amdgcn_exp2f(ml[u].x - mz);  // 0 for a piece without keys, whose O is 0
        L = fmaf(wt, ml[u].y, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(wt, v[u][e], o[e]);
      }
    }
  }
  so[wave][lane] = o;
  sml[wave][lane] = make_float2(M, L);
  __syncthreads();
  if (wave || row >= rows) return;
#pragma unroll
  for (int v = 1; v < 4; ++v) M = fmaxf(M, sml[v][lane].x);
  const float mz = M == -INFINITY ? 0.0f : M;
  L = 0.0f;
  o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float2 ml = sml[v][lane];
    const float wt = __builtin_amdgcn_exp2f(ml.x - mz);
    L = fmaf(wt, ml.y, L);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(wt, so[v][lane][e], o[e]);
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  const int sq = ar_div(row, a.g_magic);
  *reinterpret_cast<u32x2*>(a.out + ((int64_t(b) * a.win.S + sq) * a.Hq + kvh * a.G + (row - sq * a.G)) * HD + dt * 16 + g * 4) =
      u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------------- host
// Waves of a workgroup, for items of n keys at most.  us called / replayed in a graph,
// 32 query heads over 4 kv heads:
//  - 4 where they take all keys in one step, and no merge (1 row of 200, 4 / 8 waves:
//    bf16 6.9 / 7.3, 4 bits 5.7 / 6.1);
//  - 8 and no merge for a few more keys: up to 1024 of 4 bits (1 row of 800, one launch 9.4 /
//    9.3, two 11.1 / 7.9), up to 512 of bf16, and 512 more where the items alone take half
//    of the CUs (32 rows of 1500 in 4 bits, one launch 11.8, two 13.4; bf16, 24 rows of 600
//    12.0 / 14.3, 32 of 1020 16.4 / 18.1; but 16 rows of 1500 in 4 bits 11.3 / 10.8);
//  - 1, of a tile each, for few keys of bf16, whose bytes a CU takes in at its own rate (1
//    row of 500, 8 waves / 1: 9.8 / 7.5, of 380 8.0 / 7.7 and 1.3 us more on the host; window
//    of 512 + 4, 4 waves 9.9 / 2 waves 8.5 / 1 wave 7.7; but 1 row of 4000 9.3 / 8.6 / 9.6);
//  - 2, of a step each, while that is up to eight workgroups a CU in bf16 (24 rows with a
//    window of 1020, 4 / 2 waves: 16.9 / 14.7, 12 with one of 2000 15.0 / 14.4, 1 row of 4000
//    9.3 / 8.6; but 16 rows of 8000 slower) and two waves in 4 bits (1 row of 2000 8.4 / 7.9,
//    4 of 2048 8.2 / 7.7; but 8 of 1500 8.8 / 9.2), and the merge has 32 or 16 records;
//  - 4 with long runs past that.
static int as_waves(bool four, int64_t items, int64_t n, int64_t cus) {
  const int64_t tiles = (n + AS_TILE - 1) / AS_TILE, work = items * tiles;
  if (tiles <= 4) return 4;
  const bool spread = !four && tiles <= 20 && 2 * work <= 3 * cus;
  const int64_t one = 512 * ((four ? 2 : 1) + (2 * items >= cus));
  if (n <= one && items <= cus && !(spread && tiles > 6)) return 8;
  if (spread) return 1;
  return items < cus && work < (four ? 2 : 8) * cus && tiles <= (four ? 32 : 64) ? 2 : 4;
}

static AsArgs as_args(bool four, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t S_max, int64_t max_ctx,
                      int64_t window, int64_t sink, int64_t* grid) {
  AsArgs a{};
  const int64_t G = Hq / Hkv;
  a.win = win_args(S, S_max, max_ctx, window, sink);
  a.B = int(B);
  a.Hq = int(Hq);
  a.Hkv = int(Hkv);
  a.G = int(G);
  a.rts = int((S * G + AS_ROWS - 1) / AS_ROWS);
  a.g_magic = ar_magic(uint32_t(G));
  // an item's keys at most: the windows of its queries, and the gap's alignment
  const int64_t seen = int64_t(a.win.window) + a.win.sink + std::min<int64_t>(S, AS_ROWS) - 1 + (four ? 3 : 0);
  const int64_t n = std::max<int64_t>(std::min(max_ctx, seen), 1);
  const int64_t items = B * Hkv * a.rts, cus = std::max(current_device_cus(), 1);
  a.waves = as_waves(four, items, n, cus);
  const int64_t step = a.waves * AS_TILE, steps = (n + step - 1) / step;
  // Else runs for a workgroup a CU, or for two where the rows are likely of different
  // lengths and a step takes little from memory (8 rows of up to 32000 in 4 bits, 8 / 16
  // runs an item: 29.5 / 25.6 us; one row of 32000, 64 / 125 runs: 13.1 / 16.1; bf16, 32 rows
  // with a window of 8000, 2 / 4 runs: 69 / 74), but no runs of a few steps where the
  // items alone fill the CUs (64 rows of 2000 in 4 bits, 1 / 2 runs: 16.7 / 20.0).
  const int64_t places = cus * (four && B > 1 ? 2 : 1);
  int64_t want = a.waves == 8 || (items >= cus && steps <= 8) ? 1 : std::max<int64_t>(places / items, 1);
  if (a.waves < AS_CUT) want = steps;
  a.run = int((steps + want - 1) / want * step);
  a.runs = int((steps * step + a.run - 1) / a.run);
  // An even share of all keys for each place once that is 16 steps and more (runs /
  // shares: 32 rows of up to 16384 47.5 / 41.8 us, 64 of 32768 150 / 138; but 64 of 4096 25.4 /
  // 29.6, for a share begins and ends inside items).
  a.wgs = four && B > 1 && items < 4 * places && items * steps >= 16 * places ? int(places) : 0;
  *grid = a.wgs ? a.wgs : items * a.runs;
  return a;
}

// Whether rows go as streams: up to 64 of a (sequence, kv head), and more while that is
// at most four steps a CU in all.  A stream's 16 rows take nearly twice as long over many
// keys as their share of a tile's 128, but end sooner over few (1 x 100 queries on 1000
// entries in 4 bits, tiles / streams: 15.4 / 10.4 us; 8 x 12 with a window of 512 14.5 /
// 12.3; but 8 x 24 16.2 / 17.5, a prompt of 640 with a window of 250 14.5 / 21.5).  The bound
// is where the windowed ones cross.  In 4 bits there are shapes on both sides past it: 4 x
// 301 queries on 2900 (28 x the bound) 87 / 124, 4 x 100 on 1422 28.0 / 33.1, 6 x 46 on 1203
// 23.2 / 24.4, but 1 x 200 on 1000 (1.6 x) 18.0 / 14.0, 1 x 392 on 392 16.7 / 14.4, 8 x 24 on
// 2000 (3 x) 25.0 / 23.0.
static bool as_few(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t max_ctx, int64_t window,
                   int64_t sink) {
  const int64_t rows = S * (Hq / Hkv), items = B * Hkv * ((rows + AS_ROWS - 1) / AS_ROWS);
  const int64_t seen = std::min<int64_t>(window, WIN_NONE) + std::min<int64_t>(sink, WIN_NONE);
  const int64_t keys = window ? std::min(max_ctx, seen) : max_ctx;
  return rows <= 64 || items * ((keys + AS_STEP - 1) / AS_STEP) <= 4 * std::max(current_device_cus(), 1);
}
static int64_t as_bytes(const AsArgs& a) {
  const int64_t records = a.wgs ? 2 * int64_t(a.wgs) : a.runs > 1 ? int64_t(a.runs) * a.B * a.Hkv * a.rts : 0;
  return records * AS_REC * int64_t(sizeof(float));
}

template <bool FOUR>
static int as_launch(const char* fn, const AsArgs& a, hipStream_t s) {
  const dim3 g{unsigned(a.Hkv), unsigned(a.B), unsigned(a.runs * a.rts)};
  const dim3 merge{unsigned(a.Hkv * 8), unsigned(a.B), unsigned(a.rts)};
  if (a.wgs)
    hipLaunchKernelGGL(attn_stream_cut_kernel, dim3(unsigned(a.wgs)), dim3(AS_CUT * 64), 0, s, a);
  else if (a.waves == 8)
    hipLaunchKernelGGL((attn_stream_kernel<FOUR, 8>), g, dim3(512), 0, s, a);
  else if (a.waves == AS_CUT)
    hipLaunchKernelGGL((attn_stream_kernel<FOUR, AS_CUT>), g, dim3(AS_CUT * 64), 0, s, a);
  else if (a.waves == 2)
    hipLaunchKernelGGL((attn_stream_kernel<FOUR, 2>), g, dim3(128), 0, s, a);
  else
    hipLaunchKernelGGL((attn_stream_kernel<false, 1>), g, dim3(64), 0, s, a);
  const int rc = hip_status(fn);
  if (rc || (a.wgs == 0 && a.runs == 1)) return rc;
  if (a.wgs)
    hipLaunchKernelGGL((attn_stream_merge_kernel<true, true>), merge, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((attn_stream_merge_kernel<FOUR, false>), merge, dim3(256), 0, s, a);
  return hip_status(fn);
}

}  // namespace qmoe

using namespace qmoe;

// Both caches' calls, whose arguments but these are checked.
static int attend(const char* fn, bool four, const qmoe_bf16* q, const qmoe_bf16* k, const qmoe_bf16* v,
                  const Cache4& cache, const int32_t* ctx_len, int64_t B, int64_t S, int64_t Hq, int64_t Hkv,
                  int64_t S_max, int64_t max_ctx, int64_t window, int64_t sink, float scale, void* workspace,
                  int64_t workspace_bytes, qmoe_bf16* out, qmoe_stream_t stream) {
  if (B == 0 || S == 0) return QMOE_OK;
  QMOE_REQUIRE(aligned16(k, v, cache.k, cache.ks, cache.v, cache.vs), "%s: operands must be 16-byte aligned", fn);
  if (!as_few(B, S, Hq, Hkv, max_ctx, window, sink))
    return attn_window_tiles(fn, q, k, v, four ? &cache : nullptr, ctx_len, B, S, Hq, Hkv, S_max, max_ctx, window, sink,
                             scale, workspace, workspace_bytes, out, as_stream(stream));
  int64_t grid;
  AsArgs a = as_args(four, B, S, Hq, Hkv, S_max, max_ctx, window, sink, &grid);
  if (int rc = win_operands(fn, grid, as_bytes(a), workspace, workspace_bytes, q, out, B * S * Hq)) return rc;
  a.q = q;
  a.k = k;
  a.v = v;
  a.c = cache;
  a.win.ctx_len = ctx_len;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = static_cast<float*>(workspace);
  a.out = out;
  return four ? as_launch<true>(fn, a, as_stream(stream)) : as_launch<false>(fn, a, as_stream(stream));
}

static int64_t workspace(const char* fn, bool four, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                         int64_t window, int64_t sink, int64_t max_ctx) {
  const int64_t most = 1ll << 22;
  if (win_check(fn, B, S, Hq, Hkv, D, most, max_ctx, window, sink, 1.0f)) return -1;
  if (B == 0 || S == 0) return 0;
  if (!as_few(B, S, Hq, Hkv, max_ctx, window, sink))
    return attn_window_tiles_workspace(B, S, Hq, Hkv, max_ctx, window, sink);
  int64_t grid;
  return as_bytes(as_args(four, B, S, Hq, Hkv, most, max_ctx, window, sink, &grid));
}

extern "C" int64_t qmoe_attn_window_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                                              int64_t sink, int64_t max_ctx) {
  return window <= 0 ? -1 : workspace("qmoe_attn_window_workspace", false, B, S, Hq, Hkv, D, window, sink, max_ctx);
}

extern "C" int qmoe_attn_window(const qmoe_bf16* q, const qmoe_bf16* k_cache, const qmoe_bf16* v_cache,
                                const int32_t* ctx_len, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                int64_t S_max, int64_t max_ctx, int64_t window, int64_t sink, float scale,
                                void* workspace, int64_t workspace_bytes, qmoe_bf16* out, qmoe_stream_t stream) {
  const char* fn = "qmoe_attn_window";
  QMOE_REQUIRE(B == 0 || S == 0 || (q && k_cache && v_cache && ctx_len && out), "%s: null pointer", fn);
  if (int rc = win_check(fn, B, S, Hq, Hkv, D, S_max, max_ctx, window, sink, scale)) return rc;
  QMOE_REQUIRE(window > 0, "%s: window must be positive", fn);
  return attend(fn, false, q, k_cache, v_cache, Cache4{}, ctx_len, B, S, Hq, Hkv, S_max, max_ctx, window, sink, scale,
                workspace, workspace_bytes, out, stream);
}

extern "C" int64_t qmoe_attn_kv4_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                                           int64_t sink, int64_t max_ctx) {
  return workspace("qmoe_attn_kv4_workspace", true, B, S, Hq, Hkv, D, window, sink, max_ctx);
}

extern "C" int qmoe_attn_kv4(const qmoe_bf16* q, const uint8_t* k_cache, const uint8_t* k_scales,
                             const uint8_t* v_cache, const uint8_t* v_scales, const int32_t* ctx_len, int64_t B,
                             int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t S_max, int64_t max_ctx,
                             int64_t window, int64_t sink, float scale, void* workspace, int64_t workspace_bytes,
                             qmoe_bf16* out, qmoe_stream_t stream) {
  const char* fn = "qmoe_attn_kv4";
  QMOE_REQUIRE(B == 0 || S == 0 || (q && k_cache && k_scales && v_cache && v_scales && ctx_len && out),
               "%s: null pointer", fn);
  if (int rc = win_check(fn, B, S, Hq, Hkv, D, S_max, max_ctx, window, sink, scale)) return rc;
  return attend(fn, true, q, nullptr, nullptr, Cache4{k_cache, k_scales, v_cache, v_scales}, ctx_len, B, S, Hq, Hkv,
                S_max, max_ctx, window, sink, scale, workspace, workspace_bytes, out, stream);
}
