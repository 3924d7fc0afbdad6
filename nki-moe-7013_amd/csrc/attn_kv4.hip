// Attention over a cache in 4 bits (head_dim 128): few query rows over many keys,
// where the cache's stream is what costs.  Many rows go to the tiles of attn_rows.hip.
//
// A wave takes 64 keys at a time and up to 16 packed query rows (query-major, then
// the G = Hq / Hkv heads of the group), on v_mfma_f32_16x16x32_bf16:
//   S^T [keys x rows] = K . Q^T     O^T [dims x rows] += V^T . P^T
// Numbers become bf16 in registers (v_cvt_scalef32_pk_bf16_fp4, two a step with their
// power; exact), so queries and products are those of a bf16 cache.
#include "attn_tile.hpp"
#include "common.hpp"
#include "kv4.hpp"
#include "window.hpp"

namespace qmoe {

constexpr int K4_ROWS = 16;             // query rows of an item
constexpr int K4_TILE = 64;             // keys of a wave's step
constexpr int K4_STEP = 4 * K4_TILE;    // keys of a workgroup's step
constexpr int K4_MAX_ROWS = 64;         // rows of a (sequence, kv head): past them tiles share the keys
constexpr int K4_REC = 2 * K4_ROWS + K4_ROWS * HD;  // a run's record: (m, l) of the rows, O in register order

struct K4Args {
  const uint16_t* q;
  Cache4 c;
  WinArgs win;
  int B, Hq, Hkv, rts, runs, run;  // row tiles; runs of `run` steps
  uint32_t g_magic;
  float scale_log2;
  float* part;  // [runs][B * Hkv * rts][K4_REC], when runs > 1
  uint16_t* out;
};

// The keys that an item's queries see, from its first row r0 to its last, r1.  The gap
// begins at a multiple of 4, so that four keys from a multiple of 4 on are rows in a
// row; the run's rows [stay, hid) are then some that no query sees.
struct K4Run {
  WinRow first, last;
  Gap gap;
  int stay, hid, n;
};
__device__ __forceinline__ K4Run k4_run(const K4Args& a, int b, int r0, int r1) {
  K4Run k;
  k.first = win_row(a.win, b, ar_div(r0, a.g_magic));
  k.last = win_row(a.win, b, ar_div(r1, a.g_magic));
  k.stay = min(a.win.sink, k.last.end);
  const int at = (k.stay + 3) & ~3;
  k.gap = Gap{at, max(k.first.low - at, 0)};
  k.n = k.first.low <= at ? k.last.end : at + max(k.last.end - k.first.low, 0);
  k.hid = k.first.low <= at ? max(k.first.low, k.stay) : at;
  return k;
}

// A wave's 64 keys as they lie in memory.  Lane (r = lane % 16, g = lane / 16) holds
// block g of the keys 4 r + [0, 4), whose powers are 16 bytes in a row.
struct K4Tile {
  u32x4 k[4], ks, v[4], vs;
};

// V passes through LDS in bf16, row = key, 256 bytes; the pair p of 16-byte chunks sits
// at p ^ (((key ^ key / 4) % 4) + 4 (key / 16 % 2)), so that 8 lanes' writes (keys
// 4 r + j of 8 consecutive r) and a half-wave's transposing reads (keys 16 g + [0, 4)
// of two g) fall into eight different places.
__global__ __launch_bounds__(256, 2) void attn_kv4_kernel(const K4Args a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4][K4_TILE * AP_ROWB];
  __shared__ float2 sml[4][K4_ROWS];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int G = a.Hq / a.Hkv, rows = a.win.S * G, grp = a.B * a.Hkv;
  // (sequence, kv head) fastest, so the row tiles that share its keys are on one XCD
  // when their number is a multiple of 8
  const int x = int(blockIdx.x), z = x % grp, y = x / grp, rt = y % a.rts, run = y / a.rts;
  const int b = z / a.Hkv, kvh = z % a.Hkv, r0 = rt * K4_ROWS, r1 = min(r0 + K4_ROWS, rows) - 1;
  const K4Run kr = k4_run(a, b, r0, r1);
  const Gap gap = kr.gap;
  const int k0 = run * a.run * K4_STEP, k1 = min(kr.n, k0 + a.run * K4_STEP);
  if (run > 0 && k0 >= k1) return;  // the merge knows how many runs there are
  const int row = min(r0 + r, r1), sq = ar_div(row, a.g_magic);
  const bool live = r0 + r <= r1;
  const int64_t qrow = (int64_t(b) * a.win.S + sq) * a.Hq + kvh * G + (row - sq * G);
  // this lane's row sees the keys [0, stay) and [all, ...) up to row own.end
  const WinRow own = win_row(a.win, b, sq);
  const int all = own.low <= a.win.sink ? 0 : gap.key(own.low);
  // every row of the item sees the keys [from, upto)
  const int from = kr.last.low <= a.win.sink ? 0 : gap.key(kr.last.low), upto = gap.key(kr.first.end - 1) + 1;
  const int64_t base = (int64_t(b) * a.Hkv + kvh) * a.win.S_max;

  // Q^T as B operands in the order of the K blocks: step ks of lane (r, g) holds dims
  // 32 g + 8 ks + [0, 8) of row r
  bf16x8 qf[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) {
    const u32x4 w = live ? ld16(a.q + qrow * HD + g * 32 + ks * 8) : u32x4{0u, 0u, 0u, 0u};
    qf[ks] = __builtin_bit_cast(bf16x8, w);
  }
  f32x4 o[8];  // O^T: dims 16 dt + 4 g + [0, 4) of row r
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  if (k0 < k1) {
    // rows that may be read; past them numbers and powers are zeros
    const int top = min(gap.row(k1 - 1) + 1, a.win.S_max);
    const __amdgpu_buffer_rsrc_t rk = kv4_rsrc(a.c.k + base * KV4_ROWB, int64_t(top) * KV4_ROWB);
    const __amdgpu_buffer_rsrc_t rv = kv4_rsrc(a.c.v + base * KV4_ROWB, int64_t(top) * KV4_ROWB);
    const __amdgpu_buffer_rsrc_t rks = kv4_rsrc(a.c.ks + base * 4, int64_t(top) * 4);
    const __amdgpu_buffer_rsrc_t rvs = kv4_rsrc(a.c.vs + base * 4, int64_t(top) * 4);
    auto load = [&](int t0, K4Tile& t) {
      const uint32_t rr = uint32_t(gap.row(t0 + 4 * r));
#pragma unroll
      for (int j = 0; j < 4; ++j) t.k[j] = kv4_ld16(rk, (rr + j) * KV4_ROWB + g * 16);
      t.ks = kv4_ld16(rks, rr * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) t.v[j] = kv4_ld16(rv, (rr + j) * KV4_ROWB + g * 16);
      t.vs = kv4_ld16(rvs, rr * 4);
    };
    uint8_t* vt = smem[wave];
    // writes: chunk pair 2 g + c2 of key 4 r + j is in place wat[c2 ^ j]
    uint32_t wat[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      wat[i] = uint32_t(r * 4 * AP_ROWB + (((2 * g) ^ ((r & 3) | ((r >> 2) & 1) << 2)) ^ i) * 32);
    // transposing reads: 16-lane group g takes keys 16 g + 8 m + 4 h + [0, 4), dims
    // 16 dt + [0, 16), from place rat[dt ^ (2 m + h)]
    const int jr = (lane >> 2) & 3;
    uint32_t rat[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      rat[i] = uint32_t((16 * g + jr) * AP_ROWB + (i ^ (jr | (g & 1) << 2)) * 32 + (lane & 3) * 8);

    auto step = [&](int t0, const K4Tile& t) {
      f32x4 sc[4];  // S^T: keys 16 g + 4 i + j of row r
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4 c[4];
        kv4_chunks(t.k[j], kv4_scale((t.ks[j] >> (8 * g)) & 255u), c);
        sc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, c[ks]), qf[ks], sc[j], 0, 0, 0);
      }
      wave_lds_sync();  // the last tile's V reads are done
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t p = (t.vs[j] >> (8 * g)) & 255u;
        if (t0 < kr.hid && t0 + K4_TILE > kr.stay) {  // rows that no query sees add 0, whatever they hold
          const int rw = gap.row(t0 + 4 * r + j);
          p = rw >= kr.stay && rw < kr.hid ? 0u : p;
        }
        u32x4 c[4];
        kv4_chunks(t.v[j], kv4_scale(p), c);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x4*>(vt + wat[(i >> 1) ^ j] + j * AP_ROWB + (i & 1) * 16) = c[i];
      }
      if (t0 < from || t0 + K4_TILE > min(upto, k1)) {
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
    };

    // a wave's tiles wave, wave + 4, ...: the next one's loads go out before a step
    K4Tile ta, tb;
    int t0 = k0 + wave * K4_TILE;
    if (t0 < k1) load(t0, ta);
    for (; t0 < k1; t0 += 2 * K4_STEP) {
      const bool more = t0 + K4_STEP < k1;
      if (more) load(t0 + K4_STEP, tb);
      step(t0, ta);
      if (!more) break;
      if (t0 + 2 * K4_STEP < k1) load(t0 + 2 * K4_STEP, ta);
      step(t0 + K4_STEP, tb);
    }
  }

  // the waves' states of the same rows: each wave joins two of the eight dim tiles
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();  // V tiles free
  float* rec = reinterpret_cast<float*>(&smem[0][0]);
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(rec + ((wave * 8 + dt) * 64 + lane) * 4) = o[dt];
  if (g == 0) sml[wave][r] = make_float2(m, l);
  __syncthreads();
  float M = -INFINITY, L = 0.0f, wt[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w][r].x);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 ml = sml[w][r];
    wt[w] = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
    L = fmaf(wt[w], ml.y, L);
  }
  float* part = a.runs > 1 ? a.part + (int64_t(run) * grp * a.rts + z * a.rts + rt) * K4_REC : nullptr;
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int dt = wave * 2 + i;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(rec + ((w * 8 + dt) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = fmaf(wt[w], v[e], sum[e]);
    }
    if (!live) continue;
    if (part)
      *reinterpret_cast<f32x4*>(part + 2 * K4_ROWS + (dt * 64 + lane) * 4) = sum;
    else
      *reinterpret_cast<u32x2*>(a.out + qrow * HD + dt * 16 + g * 4) =
          u32x2{pack_bf16x2(sum[0] * inv, sum[1] * inv), pack_bf16x2(sum[2] * inv, sum[3] * inv)};
  }
  if (part && wave == 0 && g == 0) *reinterpret_cast<float2*>(part + 2 * r) = make_float2(M, L);
}

// Joins the runs of an item's rows: workgroup = (item, dim tile), wave w takes the
// runs w, w + 4, ..., four at a time.
__global__ __launch_bounds__(256) void attn_kv4_merge_kernel(const K4Args a) {
  __shared__ f32x4 so[4][64];
  __shared__ float2 sml[4][64];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
  const int dt = int(blockIdx.x) & 7, item = int(blockIdx.x) >> 3;
  const int G = a.Hq / a.Hkv, rows = a.win.S * G;
  const int rt = item % a.rts, z = item / a.rts, b = z / a.Hkv, kvh = z % a.Hkv, r0 = rt * K4_ROWS;
  const int n = k4_run(a, b, r0, min(r0 + K4_ROWS, rows) - 1).n, per = a.run * K4_STEP;
  const int runs = max((n + per - 1) / per, 1);
  const int row = r0 + r;
  const int64_t next = int64_t(a.B) * a.Hkv * a.rts * K4_REC;
  const float* p = a.part + int64_t(item) * K4_REC;
  float M = -INFINITY, L = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (row < rows) {
    for (int i0 = wave; i0 < runs; i0 += 16) {
      float2 ml[4];
      f32x4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + 4 * u;
        const float* q = p + min(i, runs - 1) * next;
        ml[u] = *reinterpret_cast<const float2*>(q + 2 * r);
        v[u] = *reinterpret_cast<const f32x4*>(q + 2 * K4_ROWS + (dt * 64 + lane) * 4);
        if (i >= runs) ml[u] = make_float2(-INFINITY, 0.0f);
      }
      const float to = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M);
      const float mz = to == -INFINITY ? 0.0f : to, al = __builtin_amdgcn_exp2f(M - mz);
      M = to;
      L *= al;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] *= al;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = __builtin_amdgcn_exp2f(ml[u].x - mz);  // 0 for a run without keys, whose O is 0
        L = fmaf(w, ml[u].y, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(w, v[u][e], o[e]);
      }
    }
  }
  so[wave][lane] = o;
  sml[wave][lane] = make_float2(M, L);
  __syncthreads();
  if (wave || row >= rows) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) M = fmaxf(M, sml[w][lane].x);
  const float mz = M == -INFINITY ? 0.0f : M;
  L = 0.0f;
  o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 ml = sml[w][lane];
    const float wt = __builtin_amdgcn_exp2f(ml.x - mz);
    L = fmaf(wt, ml.y, L);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(wt, so[w][lane][e], o[e]);
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  const int sq = ar_div(row, a.g_magic);
  *reinterpret_cast<u32x2*>(a.out + ((int64_t(b) * a.win.S + sq) * a.Hq + kvh * G + (row - sq * G)) * HD + dt * 16 + g * 4) =
      u32x2{pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv)};
}

// ---------------------------------------------------------------------- host
static K4Args k4_args(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t S_max, int64_t max_ctx, int64_t window,
                      int64_t sink, int64_t* grid) {
  K4Args a{};
  const int64_t G = Hq / Hkv;
  a.win = win_args(S, S_max, max_ctx, window, sink);
  a.B = int(B);
  a.Hq = int(Hq);
  a.Hkv = int(Hkv);
  a.rts = int((S * G + K4_ROWS - 1) / K4_ROWS);
  a.g_magic = ar_magic(uint32_t(G));
  // a run's keys at most: with the gap's alignment, and the windows of a tile's queries
  const int64_t n = std::min<int64_t>(max_ctx, int64_t(a.win.window) + a.win.sink + 3 + std::min<int64_t>(S, K4_ROWS)) + 3;
  const int64_t items = B * Hkv * a.rts, steps = (n + K4_STEP - 1) / K4_STEP;
  const int64_t want = std::max<int64_t>(8 * std::max(current_device_cus(), 1) / items, 1);
  a.run = int((steps + want - 1) / want);
  a.runs = int((steps + a.run - 1) / a.run);
  *grid = items * a.runs;
  return a;
}
static int64_t k4_bytes(const K4Args& a) {
  return a.runs > 1 ? int64_t(a.runs) * a.B * a.Hkv * a.rts * K4_REC * int64_t(sizeof(float)) : 0;
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int64_t qmoe_attn_kv4_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t window,
                                           int64_t sink, int64_t max_ctx) {
  const int64_t most = 1ll << 22;
  if (win_check("qmoe_attn_kv4_workspace", B, S, Hq, Hkv, D, most, max_ctx, window, sink, 1.0f)) return -1;
  if (B == 0 || S == 0) return 0;
  if (S * (Hq / Hkv) > K4_MAX_ROWS) return attn_kv4_tiles_workspace(B, S, Hq, Hkv, max_ctx, window, sink);
  int64_t grid;
  return k4_bytes(k4_args(B, S, Hq, Hkv, most, max_ctx, window, sink, &grid));
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
  if (B == 0 || S == 0) return QMOE_OK;
  QMOE_REQUIRE(aligned16(k_cache, k_scales, v_cache, v_scales), "%s: operands must be 16-byte aligned", fn);
  const Cache4 cache{k_cache, k_scales, v_cache, v_scales};
  if (S * (Hq / Hkv) > K4_MAX_ROWS)
    return attn_kv4_tiles(fn, q, cache, ctx_len, B, S, Hq, Hkv, S_max, max_ctx, window, sink, scale, workspace,
                          workspace_bytes, out, as_stream(stream));
  int64_t grid;
  K4Args a = k4_args(B, S, Hq, Hkv, S_max, max_ctx, window, sink, &grid);
  if (int rc = win_operands(fn, grid, k4_bytes(a), workspace, workspace_bytes, q, out, B * S * Hq, true)) return rc;
  a.q = q;
  a.c = cache;
  a.win.ctx_len = ctx_len;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part = static_cast<float*>(workspace);
  a.out = out;
  hipLaunchKernelGGL(attn_kv4_kernel, dim3(unsigned(grid)), dim3(256), 0, as_stream(stream), a);
  if (int rc = hip_status(fn)) return rc;
  if (a.runs == 1) return QMOE_OK;
  hipLaunchKernelGGL(attn_kv4_merge_kernel, dim3(unsigned(B * Hkv * a.rts * 8)), dim3(256), 0, as_stream(stream), a);
  return hip_status(fn);
}
