// Attention over a cache whose first part a batch shares, and causal attention
// that also accumulates each cache entry's attention weight (head_dim 128).
//
// Query rows are packed: row r of a (batch, kv head) pair is query r / G, head
// r % G of the GQA group (G = Hq / Hkv), so a 128-row tile reads each key of
// the kv head once for all of its heads.  Softmax over a concatenation of key
// runs is associative: a run leaves (m, l, O) with m its maximum, l = sum
// 2^(s - m) and O = sum 2^(s - m) v; runs join as m = max m_i, l = sum
// 2^(m_i - m) l_i, O likewise.
//
//  attn_rows_kernel   work items of (row tile, key run) over flash_segment.
//                     Decode (S * G < 128): the prefix is attended by tiles of
//                     packed rows that span the batch, so its keys are read
//                     once for every 128 of all B * S * G rows instead of once
//                     for each sequence; each sequence's own keys are items of
//                     their own.  Chunks (S * G >= 128): a tile's rows belong
//                     to one sequence and its item runs over the prefix, then
//                     over its own keys.
//  attn_rows_merge_kernel  joins the runs of a row where there are several.
//  attn_colsum_kernel      w = 2^(s - lse) summed over query rows: the scores
//                          of a key run against streamed query tiles, after
//                          the attention left each row's lse = m + log2 l.
#include "attn_tile.hpp"
#include "common.hpp"

#include <math.h>

namespace qmoe {

// Record of a run of 32 rows: (m, l) of each row, then O in register order: chunk
// (db, g) holds 4 dims (32 db + 8 g + 4 (lane / 32)) of every lane, so a store
// (and the merge's load) covers 1 KB of contiguous memory.  Rows stored one
// after another cost the merge of 20480 rows x 3 runs 11.6 us instead of 6.
constexpr int AR_REC = 64 + 16 * 64 * 4;
constexpr int AR_MAX_G = 16;      // q heads per kv head
constexpr int64_t AR_MAX_KEYS = 1ll << 22;  // keys of one run are addressed with 32-bit byte offsets

// A kind of item: `rows` query rows and runs of `run` steps of `keys` keys.
// Tiles (128 rows, 64 keys: flash_segment) share each key among four waves'
// rows; streams (32 rows, 256 keys: stream_segment) share each row among four
// waves' keys.
// `split` streams of one step keep their waves' 64 keys apart, as records of their
// own, where the join of the waves (five barriers) is longer than four records
// are for the merge.
struct ArKind {
  int stream, rts, runs, run, split;
  __host__ __device__ int records() const { return split ? 4 * runs : runs; }
  __host__ __device__ int rows() const { return stream ? 32 : 128; }
  __host__ __device__ int keys() const { return stream ? 4 * AP_KT : AP_KT; }
};

struct ArArgs {
  const uint16_t *q, *kp, *vp, *k, *v;
  const int32_t* ctx_len;  // own entries that a row's query 0 sees; nullptr: start + 1 for every row
  const int32_t* lengths;  // queries of a row that count in lse; nullptr: all
  int P, Pmax, B, S, Hq, Hkv, S_max, max_ctx, start;
  uint32_t g_magic;        // ar_magic(G)
  float scale_log2;
  uint16_t* out;
  float* part;  // when NS > 1: [pre.runs][Hkv][nb_pre][AR_REC], [own.runs][B * Hkv][nb_own][AR_REC]
  float* lse;   // [B][Hkv][S * G] or nullptr
  // n_pre prefix items (pre.rts row tiles over all B * S * G rows x pre.runs x
  // Hkv), then items of (own.rts row tiles x own.runs x B x Hkv), whose steps
  // start with the prefix when joint.  NS = pre.records() + own.records() a row.
  int NS, n_pre, joint, nb_pre, nb_own;  // nb: blocks of 32 rows
  ArKind pre, own;
};

// r / G for 0 <= r < 2^32 / G, by a multiplication
__host__ __device__ __forceinline__ uint32_t ar_magic(uint32_t G) {
  return G == 1 ? 0u : uint32_t(((1ull << 32) + G - 1) / G);
}
__device__ __forceinline__ int ar_div(uint32_t r, uint32_t magic) { return int(magic ? __umulhi(r, magic) : r); }

// Own entries that query s of batch row b sees.
__device__ __forceinline__ int ar_sees(const ArArgs& a, int b, int s) {
  const int c = a.ctx_len ? min(a.ctx_len[b], a.S_max) : a.start + 1;
  return max(min(c + s, min(a.max_ctx, a.S_max)), 0);
}

__device__ __forceinline__ float ar_lse(float m, float l) { return l > 0.0f ? m + __log2f(l) : INFINITY; }

template <bool stream>
__device__ __forceinline__ void ar_item(const ArArgs& a, const ArKind kd, const bool pre, uint8_t* smem) {
  const int lane = threadIdx.x & 63, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6);
  const int G = a.Hq / a.Hkv;
  constexpr int KS = stream ? 4 * AP_KT : AP_KT, ROWS = stream ? 32 : 128;
  const int nP = (a.P + KS - 1) / KS;  // steps of the prefix
  int kvh, b = 0, r0, rows, run;
  if (pre) {
    // (kv head, run) fastest: the row tiles of one run sit Hkv * runs items apart,
    // on one XCD (and its L2) when that is a multiple of 8
    const int grp = a.Hkv * kd.runs, x = int(blockIdx.x), y = x % grp;
    kvh = y % a.Hkv;
    run = y / a.Hkv;
    r0 = x / grp * ROWS;
    rows = a.B * a.S * G;
  } else {
    // latest row tile (the most keys) first
    const int grp = a.B * a.Hkv, x = int(blockIdx.x) - a.n_pre, y = x % (grp * kd.runs), z = y % grp;
    run = y / grp;
    b = z / a.Hkv;
    kvh = z % a.Hkv;
    r0 = (kd.rts - 1 - x / (grp * kd.runs)) * ROWS;
    rows = a.S * G;
  }
  const int off = pre || a.joint ? nP : 0;  // own steps start here
  // own keys that the tile's last row sees; the item's steps [t0, t1)
  const int seen = pre ? 0 : ar_sees(a, b, ar_div(min(r0 + ROWS, rows) - 1, a.g_magic));
  const int t0 = run * kd.run, t1 = min(off + (seen + KS - 1) / KS, t0 + kd.run);
  const int rw = r0 + (stream ? 0 : wave * 32);    // the wave's first row
  const int row = rw + (lane & 31);                // this lane's row
  const bool live = row < rows, wlive = rw < rows;
  const int rq = live ? row : rows - 1;            // a row to take the limits of
  const int sq = ar_div(rq, a.g_magic);            // its query (over the whole batch for prefix items)
  const int64_t qrow = (pre ? int64_t(sq) : int64_t(b) * a.S + sq) * a.Hq + kvh * G + (rq - sq * G);
  FlashRows st;
  st.start(live ? a.q + qrow * HD : nullptr, hl);
  // the prefix steps of the run, then its own steps (one copy of the loop's code)
#pragma unroll 1
  for (int seg = 0; seg < 2; ++seg) {
    const uint16_t *kk = a.kp, *vv = a.vp;
    int64_t base;
    int n, lim, first = -1, last = -1;
    if (seg == 0) {
      const int e = min(t1, off);
      if (t0 >= e) continue;
      const int k0 = t0 * KS;
      n = min(a.P, e * KS) - k0;
      base = (int64_t(kvh) * a.Pmax + k0) * HD;
      lim = first = n - 1;
      if (wlive) last = n - 1;
    } else {
      const int s0 = max(t0, off) - off, s1 = t1 - off;
      if (s0 >= s1) break;
      const int k0 = s0 * KS, end = min(seen, s1 * KS);
      n = end - k0;
      kk = a.k;
      vv = a.v;
      base = ((int64_t(b) * a.Hkv + kvh) * a.S_max + k0) * HD;
      lim = min(ar_sees(a, b, sq), end) - 1 - k0;
      if (wlive) {
        first = min(ar_sees(a, b, ar_div(rw, a.g_magic)), end) - 1 - k0;
        last = min(ar_sees(a, b, ar_div(min(rw + 31, rows - 1), a.g_magic)), end) - 1 - k0;
      }
    }
    if constexpr (stream)
      stream_segment(smem, kk + base, vv + base, n, lim, a.scale_log2, st);
    else
      flash_segment(smem, kk + base, vv + base, n, lim, __builtin_amdgcn_readfirstlane(first),
                    __builtin_amdgcn_readfirstlane(last), a.scale_log2, st);
  }
  if (stream && !kd.split) {
    flash_join(smem, st);
    if (wave) return;
  }
  const int rec_run = stream && kd.split ? run * 4 + wave : run;
  const float l = st.row_sum();
  if (!live) return;
  if (a.NS > 1) {
    const int64_t blk = pre ? (int64_t(rec_run) * a.Hkv + kvh) * a.nb_pre + rw / 32
                            : int64_t(a.pre.records()) * a.Hkv * a.nb_pre +
                                  ((int64_t(rec_run) * a.B + b) * a.Hkv + kvh) * a.nb_own + rw / 32;
    float* rec = a.part + blk * AR_REC;
    if (hl == 0) *reinterpret_cast<float2*>(rec + (lane & 31) * 2) = make_float2(st.m, l);
#pragma unroll
    for (int c = 0; c < 16; ++c)
      *reinterpret_cast<float4*>(rec + 64 + (c * 64 + lane) * 4) =
          make_float4(st.o[c >> 2][(c & 3) * 4], st.o[c >> 2][(c & 3) * 4 + 1], st.o[c >> 2][(c & 3) * 4 + 2],
                      st.o[c >> 2][(c & 3) * 4 + 3]);
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  uint16_t* op = a.out + qrow * HD;
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u32x2 w;
      w.x = pack_bf16x2(st.o[db][g * 4 + 0] * inv, st.o[db][g * 4 + 1] * inv);
      w.y = pack_bf16x2(st.o[db][g * 4 + 2] * inv, st.o[db][g * 4 + 3] * inv);
      *reinterpret_cast<u32x2*>(op + db * 32 + g * 8 + hl * 4) = w;
    }
  if (a.lse && hl == 0 && !pre)
    a.lse[(int64_t(b) * a.Hkv + kvh) * rows + row] =
        a.lengths && sq >= a.lengths[b] ? INFINITY : ar_lse(st.m, l);
}

// Both kinds of item in one launch: the prefix's tiles are bound by the matrix
// pipe beside the softmax's VALU work (two causal prompts of 4096: 300 us, 0.92
// PFLOP/s), the streams by their waves' chains, a loaded round trip and then the
// MFMAs and the softmax of each 64-key tile (32 rows on 8192 + up to 512 entries:
// 20 us, four tiles a wave of the prefix and one of the own entries; the 134 MB come
// at 6.6 TB/s, of the 37 that the L2s deliver), and they share the CUs (64 rows on
// 32768 + up to 1024: 60 us).
template <bool TILES, bool STREAMS>
__global__ __launch_bounds__(256, 2) void attn_rows_kernel(const ArArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[FL_SMEM];
  const bool pre = int(blockIdx.x) < a.n_pre;
  const ArKind kd = pre ? a.pre : a.own;
  if constexpr (TILES && STREAMS) {
    if (kd.stream)
      ar_item<true>(a, kd, pre, smem);
    else
      ar_item<false>(a, kd, pre, smem);
  } else {
    ar_item<STREAMS>(a, kd, pre, smem);
  }
}

// Joins the runs of 32 packed rows of a kv head (8 x 101 queries, 2 runs, 8 us; 64
// rows, 21 runs, 6.5): a chunk (db, g) of their dims
// a wave, from every record; the prefix's records hold the same 32 rows, the own
// ones those of each row's sequence.  WAVES_A_CHUNK = 1: workgroup y takes the
// four chunks of block db = y.  4: it takes chunk y alone, each wave every fourth
// run (few rows with many runs: one row of waves would wait for one load after
// another), and the waves' (m, l, O) join in LDS in wave order.
constexpr int AR_MANY_RUNS = 6;
template <int WAVES_A_CHUNK>
__global__ __launch_bounds__(256) void attn_rows_merge_kernel(const ArArgs a) {
  constexpr bool MANY = WAVES_A_CHUNK == 4;
  __shared__ __attribute__((aligned(16))) uint16_t tile[32][36];
  __shared__ __attribute__((aligned(16))) float red[MANY ? 4 : 1][64][4];
  __shared__ float2 rml[MANY ? 4 : 1][64];
  const int lane = threadIdx.x & 63, col = lane & 31, hl = lane >> 5, w = threadIdx.x >> 6;
  const int chunk = MANY ? int(blockIdx.y) : int(blockIdx.y) * 4 + w;
  const int G = a.Hq / a.Hkv, kvh = int(blockIdx.x) % a.Hkv, rb = int(blockIdx.x) / a.Hkv, per = a.S * G;
  const int rows = a.B * per, row = rb * 32 + col, r = min(row, rows - 1);
  const int sq = ar_div(r, a.g_magic), b = sq / a.S, rib = r - b * per;
  const int64_t pre_next = int64_t(a.Hkv) * a.nb_pre * AR_REC, own_next = int64_t(a.B) * a.Hkv * a.nb_own * AR_REC;
  const float* pp = a.part + (int64_t(kvh) * a.nb_pre + rb) * AR_REC;
  const float* po = a.part + a.pre.records() * pre_next + ((int64_t(b) * a.Hkv + kvh) * a.nb_own + rib / 32) * AR_REC;
  const int own_lane = rib % 32 + hl * 32;
  float M = -INFINITY, L = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  // four runs at a time: all their loads, then the joint maximum once
  for (int i0 = MANY ? w : 0; i0 < a.NS; i0 += 4 * WAVES_A_CHUNK) {
    float2 ml[4];
    f32x4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * WAVES_A_CHUNK, j = min(i, a.NS - 1);
      const bool pre = j < a.pre.records();
      const float* p = pre ? pp + j * pre_next : po + (j - a.pre.records()) * own_next;
      const int ln = pre ? lane : own_lane;
      ml[u] = *reinterpret_cast<const float2*>(p + (ln & 31) * 2);
      v[u] = *reinterpret_cast<const f32x4*>(p + 64 + (chunk * 64 + ln) * 4);
      if (i >= a.NS) ml[u] = make_float2(-INFINITY, 0.0f);
    }
    const float m = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), M), mz = m == -INFINITY ? 0.0f : m;
    const float al = __builtin_amdgcn_exp2f(M - mz);
    M = m;
    L *= al;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= al;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float wt = __builtin_amdgcn_exp2f(ml[u].x - mz);  // 0 for a run without keys, whose O is 0
      L = fmaf(wt, ml[u].y, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(wt, v[u][e], o[e]);
    }
  }
  if constexpr (MANY) {
    *reinterpret_cast<f32x4*>(red[w][lane]) = o;
    rml[w][lane] = make_float2(M, L);
    __syncthreads();
    if (w) return;
    float m = M;
#pragma unroll
    for (int i = 1; i < 4; ++i) m = fmaxf(m, rml[i][lane].x);
    const float mz = m == -INFINITY ? 0.0f : m, al = __builtin_amdgcn_exp2f(M - mz);
    L *= al;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= al;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const float wt = __builtin_amdgcn_exp2f(rml[i][lane].x - mz);
      const f32x4 v = *reinterpret_cast<const f32x4*>(red[i][lane]);
      L = fmaf(wt, rml[i][lane].y, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(wt, v[e], o[e]);
    }
    M = m;
  }
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  u32x2 pk;
  pk.x = pack_bf16x2(o[0] * inv, o[1] * inv);
  pk.y = pack_bf16x2(o[2] * inv, o[3] * inv);
  if (a.lse && chunk == 0 && hl == 0 && row < rows)
    a.lse[(int64_t(b) * a.Hkv + kvh) * per + rib] =
        a.lengths && sq - b * a.S >= a.lengths[b] ? INFINITY : ar_lse(M, L);
  if constexpr (MANY) {
    if (row < rows)
      *reinterpret_cast<u32x2*>(a.out + (int64_t(sq) * a.Hq + kvh * G + (row - sq * G)) * HD + chunk * 8 + hl * 4) = pk;
  } else {  // 64 bytes of a row at a time
    *reinterpret_cast<u32x2*>(&tile[col][w * 8 + hl * 4]) = pk;
    __syncthreads();
    const int orow = rb * 32 + int(threadIdx.x) / 8, oc = int(threadIdx.x) % 8 * 4;
    if (orow >= rows) return;
    const int oq = ar_div(orow, a.g_magic);
    *reinterpret_cast<u32x2*>(a.out + (int64_t(oq) * a.Hq + kvh * G + (orow - oq * G)) * HD + blockIdx.y * 32 + oc) =
        *reinterpret_cast<const u32x2*>(&tile[threadIdx.x / 8][oc]);
  }
}

// ====================================================================== column sums
constexpr int CS_KEYS = 256;  // keys of a workgroup (4 waves x 64)
constexpr int CS_QT = 64;     // query rows of a streamed tile
constexpr int CS_BUFS = 3, CS_LBUFS = 4;
constexpr int CS_QBYTES = CS_QT * AP_ROWB;

struct CsArgs {
  const uint16_t *q, *k;
  const float* lse;        // [B][Hkv][S * G]
  const int32_t* lengths;  // or nullptr
  int B, S, Hq, Hkv, S_max, start, n_keys, nkt, n_chunk, run;
  uint32_t g_magic;  // ar_magic(G)
  float scale_log2;
  float* part;    // [n_chunk][B][Hkv][nkt * CS_KEYS]: a sum for each run
  float* scores;  // [B][Hkv][S_max]
};

// The packed rows that see key tile kt start at (about) row cs_first, a multiple
// of CS_QT; its row tiles up to the last counted row are cut into runs of
// equal length, at most `run` tiles.  len: counted queries.
__device__ __forceinline__ int cs_first(const CsArgs& a, int kt, int G) {
  return max(kt * CS_KEYS - a.start, 0) * G / CS_QT * CS_QT;
}
__device__ __forceinline__ int cs_tiles(const CsArgs& a, int kt, int G, int len) {
  return max((len * G - cs_first(a, kt, G) + CS_QT - 1) / CS_QT, 0);
}
__device__ __forceinline__ int cs_len(const CsArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
}

// Two prompts of 4096: 190 us, 0.72 PFLOP/s, bound by one exponential a score beside
// the MFMAs.  Item (b, kv head, key tile, run of query rows): a wave keeps 64 keys as
// the B operands of S = Q . K^T, query tiles of 64 packed rows stream through
// LDS, and since lane l of a 32 x 32 block holds column l % 32, a key's sum
// over the rows of a tile is an addition within the lane.
__global__ __launch_bounds__(256, 2) void attn_colsum_kernel(const CsArgs a) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[CS_BUFS * CS_QBYTES];
  __shared__ __attribute__((aligned(1024))) float ls[CS_LBUFS][4][CS_QT];  // a copy for each wave
  const int t = threadIdx.x, lane = t & 63, hl = lane >> 5, col = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int G = a.Hq / a.Hkv, grp = a.B * a.Hkv;
  const int x = int(blockIdx.x), bh = x % grp, y = x / grp, kt = y % a.nkt, ch = y / a.nkt;
  const int b = bh / a.Hkv, kvh = bh % a.Hkv;
  const int key0 = kt * CS_KEYS;
  const int len = cs_len(a, b), tiles = cs_tiles(a, kt, G, len), runs = (tiles + a.run - 1) / a.run;
  if (ch >= runs) return;  // the addition knows how many runs a key tile has
  const int per = (tiles + runs - 1) / runs;
  const int q0 = cs_first(a, kt, G) + ch * per * CS_QT, q1 = min(q0 + per * CS_QT, len * G);
  if (q0 >= q1) {  // rounding left the last run empty
    a.part[(int64_t(ch) * grp + bh) * (int64_t(a.nkt) * CS_KEYS) + key0 + t] = 0.0f;
    return;
  }
  const int n_t = (q1 - q0 + CS_QT - 1) / CS_QT;
  // K as B operands: column block cb, k-step ks: key key0 + 64 wave + 32 cb + col
  bf16x8 kf[2][HD / 16];
  int rmin[2];  // the first packed row that sees this lane's key
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    const int key = min(key0 + wave * 64 + cb * 32 + col, a.n_keys - 1);
    rmin[cb] = max(key - a.start, 0) * G;
    const uint16_t* kp = a.k + ((int64_t(b) * a.Hkv + kvh) * a.S_max + key) * HD + hl * 8;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const u32x4 v = ld16(kp + ks * 16);
      kf[cb][ks] = __builtin_bit_cast(bf16x8, v);
    }
  }
  const int wave_rmax = max(min(key0 + wave * 64 + 63, a.n_keys - 1) - a.start, 0) * G;  // past it: no mask
  // the row (s, g) sits s * Hq + g rows after the base; rows of queries >= len read as zeros
  const pipe::i32x4 rq = pipe::make_rsrc(a.q + ((int64_t(b) * a.S) * a.Hq + kvh * G) * HD,
                                         (uint32_t(len - 1) * a.Hq + G) * AP_ROWB);
  const pipe::i32x4 rl = pipe::make_rsrc(a.lse + (int64_t(b) * a.Hkv + kvh) * (int64_t(a.S) * G),
                                         uint32_t(q1) * 4u);
  const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>(smem));
  const uint32_t lds_l = uint32_t(reinterpret_cast<uintptr_t>(&ls[0][0][0])) + uint32_t(wave * CS_QT * 4);
  auto dma_q = [&](int i) {
    const int buf = i % CS_BUFS;
    const uint32_t dst = lds0 + uint32_t(buf * CS_QBYTES + wave * 4096);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int rr = 16 * wave + 4 * j + (lane >> 4);
      const uint32_t r = uint32_t(q0 + i * CS_QT + rr);
      const int s = ar_div(r, a.g_magic), g = int(r) - s * G;
      const uint32_t off = (uint32_t(s) * a.Hq + g) * AP_ROWB + uint32_t(ap_kslot(rr, lane & 15) * 16);
      pipe::dma16(dst + j * 1024, s < len ? off : pipe::PAD, rq, 0);
    }
    pipe::dma4(lds_l + uint32_t(i % CS_LBUFS * 4 * CS_QT * 4), uint32_t(q0 + i * CS_QT + lane) * 4u, rl, 0);
  };
  float acc[2] = {0.0f, 0.0f};
  // S of rows [32 rb, 32 rb + 32) of tile i
  auto qk = [&](int i, int rb, f32x16 (&sc)[2]) {
    const uint8_t* qp = smem + i % CS_BUFS * CS_QBYTES + (rb * 32 + col) * AP_ROWB;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      const bf16x8 a0 = *reinterpret_cast<const bf16x8*>(qp + ap_kslot(lane, 2 * ks + hl) * 16);
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
        sc[cb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a0, kf[cb][ks], ks ? sc[cb] : f32x16{}, 0, 0, 0);
    }
  };
  // their weights into the sums
  auto add = [&](int i, int rb, f32x16 (&sc)[2], auto masked) {
    const int r0 = q0 + i * CS_QT + rb * 32 + hl * 4;
#pragma unroll
    for (int g4 = 0; g4 < 4; ++g4) {
      const float4 le = *reinterpret_cast<const float4*>(&ls[i % CS_LBUFS][wave][rb * 32 + g4 * 8 + hl * 4]);
      const float lo[4] = {le.x, le.y, le.z, le.w};
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float w = __builtin_amdgcn_exp2f(fmaf(sc[cb][g4 * 4 + e], a.scale_log2, -lo[e]));
          if constexpr (decltype(masked)::value) {
            const int r = r0 + g4 * 8 + e;
            w = r < rmin[cb] || r >= q1 ? 0.0f : w;
          }
          acc[cb] += w;
        }
    }
  };
  // S of one half tile is issued before the weights of the half before it
  auto step = [&](int i, int rb, f32x16 (&cur)[2], int ni, int nrb, f32x16 (&nxt)[2]) {
    const int rt = q0 + i * CS_QT;
    if (rt < wave_rmax || rt + CS_QT > q1) {
      qk(ni, nrb, nxt);
      add(i, rb, cur, std::true_type{});
    } else {
      qk(ni, nrb, nxt);
      add(i, rb, cur, std::false_type{});
    }
  };
  f32x16 sa[2], sb[2];
  dma_q(0);
  if (n_t > 1) {
    dma_q(1);
    pipe::wait_vm<5>();
  } else {
    pipe::wait_vm<0>();
  }
  __syncthreads();
  if (n_t > 2) dma_q(2);
  qk(0, 0, sa);
  for (int i = 0; i + 1 < n_t; ++i) {
    step(i, 0, sa, i, 1, sb);
    if (i + 2 < n_t)
      pipe::wait_vm<5>();
    else
      pipe::wait_vm<0>();
    __syncthreads();  // tile i + 1 visible, tile i's queries read (its lse not yet: CS_LBUFS)
    if (i + 3 < n_t) dma_q(i + 3);
    step(i, 1, sb, i + 1, 0, sa);
  }
  step(n_t - 1, 0, sa, n_t - 1, 1, sb);
  add(n_t - 1, 1, sb, std::true_type{});
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) acc[cb] += __shfl_xor(acc[cb], 32, 64);
  if (hl == 0) {
    float* pp = a.part + (int64_t(ch) * grp + bh) * (int64_t(a.nkt) * CS_KEYS) + key0 + wave * 64 + col;
    pp[0] = acc[0];
    pp[32] = acc[1];
  }
}

// scores += the runs' sums (4-5 us, one launch of round trips): a workgroup takes 64 keys, wave w the runs w, w +
// 4, ..., each eight loads at a time, and the waves' sums join in wave order.
__global__ __launch_bounds__(256) void attn_colsum_add_kernel(const CsArgs a) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int slices = a.nkt * (CS_KEYS / 64), grp = a.B * a.Hkv;
  const int bh = int(blockIdx.x) / slices, key = int(blockIdx.x) % slices * 64 + lane;
  const int c1 = (cs_tiles(a, key / CS_KEYS, a.Hq / a.Hkv, cs_len(a, bh / a.Hkv)) + a.run - 1) / a.run;
  if (c1 == 0) return;
  const float* p = a.part + int64_t(bh) * a.nkt * CS_KEYS + key;
  const int64_t next = int64_t(grp) * a.nkt * CS_KEYS;
  float sum = 0.0f;
  for (int c = wave; c < c1; c += 32) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = c + 4 * u < c1 ? p[(c + 4 * u) * next] : 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += v[u];
  }
  red[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && key < a.n_keys)
    a.scores[int64_t(bh) * a.S_max + key] += (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// ---------------------------------------------------------------------- host
static int64_t ar_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Cuts the work into items.  own_keys: own keys of a row at most.
//
// Rows of one sequence that fill a tile (S * G >= 128) run over the prefix and
// their own keys in one item.  Fewer rows leave the prefix to items of its own,
// whose rows span the batch, and take their own keys as streams (more than 64
// rows: as tiles).  The prefix goes as streams, which read its keys again for
// every 32 rows (from L2) but wait for no barrier, while that is at most
// AR_STREAM_KEYS keys in all, and as tiles past it (streams / tiles in us: 128 rows
// on 16000 keys 21.3 / 22.9, on 32768 31.4 / 30.1; 256 rows on 8192 22.4 / 24.4, on
// 32768 48.6 / 38.7; 320 rows on 3000 16.0 / 20.1; 512 rows on 1000 25.7 / 26.9, on
// 8192 31.9 / 29.1, on 32768 95 / 65).
constexpr int64_t AR_MIN_TILES = 4, AR_STREAM_KEYS = 65536;

// A tile step takes about 1.45 us with one workgroup on a CU and 2.14 with two; a
// second run costs the merge's launch, and every run a record of 528 bytes for
// each of `rows` rows (of one head), written and read at about 6 MB/us.
// Measured: 8 x 101 queries on 2900 + 101 keys, 1 run 71.7 us, 2 runs 63.6, 3 72.4;
// 512 queries on 4000 + 512 keys, 2 runs 62.7, 3 57.4, 4 53.7, 6 69.6; a 640-token
// prompt, 1 run 34.4 us, 2 38.9.
static int64_t ar_joint_runs(int64_t items, int64_t steps, int64_t rows, int64_t cus) {
  int64_t best = 1;
  double least = 1e30;
  for (int64_t n = 1; n <= 16 && n <= std::max<int64_t>(steps, 1); ++n) {
    const double step = items * n <= cus ? 1.45 : 2.14 * double(ar_ceil(items * n, 2 * cus));
    const double us = double(ar_ceil(steps, n)) * step + (n > 1 ? 4.5 + double(rows * n) * (2 * 528 / 6e6) : 0.0);
    if (us < least) {
      least = us;
      best = n;
    }
  }
  return best;
}

static void ar_cut(ArKind& kd, int64_t steps, int64_t want) {
  want = std::max<int64_t>(1, std::min(want, steps / (kd.stream ? 1 : AR_MIN_TILES)));
  kd.run = int(std::max<int64_t>(1, ar_ceil(steps, want)));
  kd.runs = int(ar_ceil(steps, kd.run));
}

static void ar_plan(ArArgs& a, int64_t own_keys, int64_t* grid) {
  const int64_t G = a.Hq / a.Hkv, rows = a.S * G, all = int64_t(a.B) * rows, groups = int64_t(a.B) * a.Hkv;
  const int64_t cus = std::max(current_device_cus(), 1);
  a.joint = rows >= 128;
  a.pre.stream = !a.joint && ar_ceil(all, 32) * a.P <= AR_STREAM_KEYS;
  a.own.stream = rows <= 64;
  a.pre.rts = int(ar_ceil(all, a.pre.rows()));
  a.own.rts = int(ar_ceil(rows, a.own.rows()));
  const int64_t pre_items = int64_t(a.pre.rts) * a.Hkv, own_items = a.own.rts * groups;
  const int64_t pre_steps = a.joint ? 0 : ar_ceil(a.P, a.pre.keys());
  const int64_t own_steps = ar_ceil(own_keys, a.own.keys()) + (a.joint ? ar_ceil(a.P, a.own.keys()) : 0);
  // Items of the prefix: one a CU (their records cost more than the CU's second
  // place gives); long runs of tiles share the CUs' two places with the own items
  // by the time of each (a tile step 1.07 us of a CU, a stream step about 5, which
  // is its share of the memory's rate).
  int64_t places = cus;
  if (!a.joint && !a.pre.stream && pre_items * pre_steps >= 8 * cus) {
    const double pre_us = 1.07 * double(pre_items * pre_steps);
    const double own_us = (a.own.stream ? 5.0 : 1.07) * double(own_items * own_steps);
    places = int64_t(2.0 * double(cus) * pre_us / (pre_us + own_us));
  }
  ar_cut(a.pre, pre_steps, places / pre_items);
  ar_cut(a.own, own_steps,
         a.joint ? ar_joint_runs(own_items, own_steps, int64_t(a.B) * a.S * a.Hq, cus) : cus / own_items);
  if (a.pre.runs + a.own.runs == 0) a.own.runs = 1;  // nothing to see: items that write zeros
  // us without and with: 4 rows on 300 + 24 keys 10.7 / 9.6, 8 rows on 300 + 250 10.7 /
  // 9.8; but 1 row on 4096 + 200 (17 runs) 11.1 / 12.1, 64 rows on 1000 + 1000 26.1 / 30.8
  const bool few = a.pre.runs + a.own.runs <= 4 && pre_items * a.pre.runs + own_items * a.own.runs <= 128;
  a.pre.split = few && a.pre.stream && a.pre.run == 1;
  a.own.split = few && a.own.stream && a.own.run == 1;
  a.NS = a.pre.records() + a.own.records();
  a.n_pre = int(pre_items * a.pre.runs);
  a.nb_pre = a.pre.runs ? int(ar_ceil(all, 32)) : 0;
  a.nb_own = a.own.runs ? int(ar_ceil(rows, 32)) : 0;
  a.g_magic = ar_magic(uint32_t(G));
  *grid = a.n_pre + own_items * a.own.runs;
}

static int64_t ar_part_bytes(const ArArgs& a) {
  if (a.NS <= 1) return 0;
  const int64_t blocks =
      int64_t(a.pre.records()) * a.Hkv * a.nb_pre + int64_t(a.own.records()) * a.B * a.Hkv * a.nb_own;
  return blocks * AR_REC * int64_t(sizeof(float));
}

static int ar_launch(const char* fn, ArArgs& a, int64_t grid, hipStream_t s) {
  const bool own = grid > a.n_pre, tiles = (a.n_pre && !a.pre.stream) || (own && !a.own.stream);
  const bool streams = (a.n_pre && a.pre.stream) || (own && a.own.stream);
  const dim3 g{unsigned(grid)}, t{256};
  if (tiles && streams)
    hipLaunchKernelGGL((attn_rows_kernel<true, true>), g, t, 0, s, a);
  else if (tiles)
    hipLaunchKernelGGL((attn_rows_kernel<true, false>), g, t, 0, s, a);
  else
    hipLaunchKernelGGL((attn_rows_kernel<false, true>), g, t, 0, s, a);
  int rc = hip_status(fn);
  if (rc || a.NS == 1) return rc;
  const int64_t blocks = ar_ceil(int64_t(a.B) * a.S * (a.Hq / a.Hkv), 32) * a.Hkv;
  if (a.NS >= AR_MANY_RUNS)
    hipLaunchKernelGGL(attn_rows_merge_kernel<4>, dim3(unsigned(blocks), 16), t, 0, s, a);
  else
    hipLaunchKernelGGL(attn_rows_merge_kernel<1>, dim3(unsigned(blocks), 4), t, 0, s, a);
  return hip_status(fn);
}

// Limits shared by both entry points; B * S may be 0.
static int ar_check(const char* fn, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t S_max,
                    float scale) {
  QMOE_REQUIRE(D == HD, "%s: head_dim must be 128 (D=%lld)", fn, (long long)D);
  QMOE_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= AR_MAX_G && Hkv < 4096,
               "%s: need Hq %% Hkv == 0, Hq / Hkv <= 16 and Hkv < 4096", fn);
  QMOE_REQUIRE(B >= 0 && B < 65536 && S >= 0 && S < (1ll << 22) && B * S * Hq < (1ll << 27),
               "%s: bad B/S (B * S * Hq must be below 2^27)", fn);
  QMOE_REQUIRE(S_max > 0 && S_max <= AR_MAX_KEYS, "%s: S_max must be in [1, 2^22]", fn);
  QMOE_REQUIRE(scale > 0.0f && std::isfinite(scale), "%s: scale must be positive and finite", fn);
  return QMOE_OK;
}

static ArArgs ar_args(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t S_max) {
  ArArgs a{};
  a.B = int(B);
  a.S = int(S);
  a.Hq = int(Hq);
  a.Hkv = int(Hkv);
  a.S_max = int(S_max);
  return a;
}

// Length of a run of row tiles in the column sums.  Two workgroups fit a CU;
// with k rounds of them the runs are about (all row tiles) / (k * places - key
// tiles) long (each key tile rounds its number of runs up), and a run costs
// about CS_START tiles more (K loads, the first tiles' round trip).
constexpr int64_t CS_START = 5;
static void cs_plan(CsArgs& a) {
  const int64_t G = a.Hq / a.Hkv, tiles = ar_ceil(a.S * G, CS_QT);
  a.nkt = int(ar_ceil(a.n_keys, CS_KEYS));
  int64_t sum = 0;  // row tiles over the key tiles of one (row, kv head)
  for (int64_t kt = 0; kt < a.nkt; ++kt) sum += tiles - std::max<int64_t>(kt * CS_KEYS - a.start, 0) * G / CS_QT;
  const int64_t places = 2 * int64_t(std::max(current_device_cus(), 1)), grp = int64_t(a.B) * a.Hkv;
  int64_t best = INT64_MAX;
  for (int64_t k = 1; k <= 8; ++k) {
    const int64_t room = k * places / grp - a.nkt;
    const int64_t run = room > 0 ? std::max<int64_t>(ar_ceil(sum, room), 1) : tiles;
    const int64_t rounds = ar_ceil(grp * (sum / run + a.nkt), places), cost = rounds * (run + CS_START);
    if (cost < best) {
      best = cost;
      a.run = int(run);
    }
  }
  a.n_chunk = int(ar_ceil(tiles, a.run));
  a.g_magic = ar_magic(uint32_t(G));
}

}  // namespace qmoe

using namespace qmoe;

extern "C" int64_t qmoe_attn_shared_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                              int64_t P, int64_t max_ctx) {
  if (B < 0 || S < 0 || P < 0 || max_ctx < 0 || max_ctx > AR_MAX_KEYS || P > AR_MAX_KEYS ||
      ar_check("qmoe_attn_shared_workspace", B, S, Hq, Hkv, D, 1, 1.0f))
    return -1;
  if (B == 0 || S == 0) return 0;
  ArArgs a = ar_args(B, S, Hq, Hkv, 1);
  int64_t grid;
  a.P = int(P);
  ar_plan(a, max_ctx, &grid);
  return ar_part_bytes(a);
}

extern "C" int qmoe_attn_shared(const qmoe_bf16* q, const qmoe_bf16* k_prefix, const qmoe_bf16* v_prefix, int64_t P,
                                int64_t P_max, const qmoe_bf16* k_cache, const qmoe_bf16* v_cache,
                                const int32_t* ctx_len, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                int64_t S_max, int64_t max_ctx, float scale, void* workspace,
                                int64_t workspace_bytes, qmoe_bf16* out, qmoe_stream_t stream) {
  const char* fn = "qmoe_attn_shared";
  QMOE_REQUIRE(B == 0 || S == 0 || (q && k_cache && v_cache && ctx_len && out), "%s: null pointer", fn);
  if (int rc = ar_check(fn, B, S, Hq, Hkv, D, S_max, scale)) return rc;
  QMOE_REQUIRE(P >= 0 && P <= P_max && P_max <= AR_MAX_KEYS, "%s: need 0 <= P <= P_max <= 2^22", fn);
  QMOE_REQUIRE(P == 0 || (k_prefix && v_prefix), "%s: null prefix", fn);
  QMOE_REQUIRE(max_ctx >= 0 && max_ctx <= S_max, "%s: need 0 <= max_ctx <= S_max", fn);
  if (B == 0 || S == 0) return QMOE_OK;
  ArArgs a = ar_args(B, S, Hq, Hkv, S_max);
  a.q = q;
  a.kp = k_prefix;
  a.vp = v_prefix;
  a.k = k_cache;
  a.v = v_cache;
  a.ctx_len = ctx_len;
  a.P = int(P);
  a.Pmax = int(P_max);
  a.max_ctx = int(max_ctx);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  a.part = static_cast<float*>(workspace);
  int64_t grid;
  ar_plan(a, max_ctx, &grid);
  QMOE_REQUIRE(grid < (1ll << 31), "%s: grid too large", fn);
  const int64_t need = ar_part_bytes(a);
  QMOE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace of %lld bytes, need %lld", fn,
               (long long)workspace_bytes, (long long)need);
  QMOE_REQUIRE(aligned16(q, k_prefix, v_prefix, k_cache, v_cache, a.part, out), "%s: operands must be 16-byte aligned",
               fn);
  return ar_launch(fn, a, grid, as_stream(stream));
}

namespace qmoe {
static void ps_plan(ArArgs& a, CsArgs& c, int64_t start, int64_t* grid) {
  a.start = int(start);
  a.max_ctx = a.S_max;
  ar_plan(a, start + a.S, grid);
  c.B = a.B;
  c.S = a.S;
  c.Hq = a.Hq;
  c.Hkv = a.Hkv;
  c.S_max = a.S_max;
  c.start = int(start);
  c.n_keys = int(start + a.S);
  cs_plan(c);
}
static int64_t ps_lse_bytes(const ArArgs& a) { return ar_ceil(int64_t(a.B) * a.S * a.Hq * 4, 256) * 256; }
static int64_t ps_col_bytes(const CsArgs& c) {
  return int64_t(c.n_chunk) * c.B * c.Hkv * c.nkt * CS_KEYS * int64_t(sizeof(float));
}
}  // namespace qmoe

extern "C" int64_t qmoe_attn_prefill_scored_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                                      int64_t start) {
  if (start < 0 || S < 0 || S > AR_MAX_KEYS || start > AR_MAX_KEYS - S ||
      ar_check("qmoe_attn_prefill_scored_workspace", B, S, Hq, Hkv, D, std::max<int64_t>(start + S, 1), 1.0f))
    return -1;
  if (B == 0 || S == 0) return 0;
  ArArgs a = ar_args(B, S, Hq, Hkv, start + S);
  CsArgs c{};
  int64_t grid;
  ps_plan(a, c, start, &grid);
  return ps_lse_bytes(a) + std::max(ar_part_bytes(a), ps_col_bytes(c));
}

extern "C" int qmoe_attn_prefill_scored(const qmoe_bf16* q, const qmoe_bf16* k_cache, const qmoe_bf16* v_cache,
                                        int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t S_max,
                                        int64_t start, const int32_t* lengths, float scale, void* workspace,
                                        int64_t workspace_bytes, float* scores, qmoe_bf16* out,
                                        qmoe_stream_t stream) {
  const char* fn = "qmoe_attn_prefill_scored";
  QMOE_REQUIRE(k_cache && v_cache && scores && (B == 0 || S == 0 || (q && out)), "%s: null pointer", fn);
  if (int rc = ar_check(fn, B, S, Hq, Hkv, D, S_max, scale)) return rc;
  QMOE_REQUIRE(start >= 0 && start <= S_max - S, "%s: need 0 <= start and start + S <= S_max", fn);
  // a row's queries are addressed with 32-bit byte offsets
  QMOE_REQUIRE(S * Hq * AP_ROWB < (1ll << 31), "%s: S * Hq must be below 2^23", fn);
  if (B == 0 || S == 0) return QMOE_OK;
  ArArgs a = ar_args(B, S, Hq, Hkv, S_max);
  CsArgs c{};
  int64_t grid;
  ps_plan(a, c, start, &grid);
  const int64_t lse = ps_lse_bytes(a), need = lse + std::max(ar_part_bytes(a), ps_col_bytes(c));
  QMOE_REQUIRE(workspace && workspace_bytes >= need, "%s: workspace of %lld bytes, need %lld", fn,
               (long long)workspace_bytes, (long long)need);
  const int64_t cgrid = int64_t(B) * Hkv * c.nkt * c.n_chunk;
  QMOE_REQUIRE(grid < (1ll << 31) && cgrid < (1ll << 31) && int64_t(B) * Hkv * c.nkt * (CS_KEYS / 64) < (1ll << 31),
               "%s: grid too large", fn);
  QMOE_REQUIRE(aligned16(q, k_cache, v_cache, static_cast<uint8_t*>(workspace), out),
               "%s: operands must be 16-byte aligned", fn);
  const uintptr_t q0 = reinterpret_cast<uintptr_t>(q), o0 = reinterpret_cast<uintptr_t>(out);
  QMOE_REQUIRE((q0 < o0 ? o0 - q0 : q0 - o0) >= uintptr_t(B * S * Hq * AP_ROWB),
               "%s: out overlaps q, which the scores read once more", fn);
  a.q = c.q = q;
  a.k = c.k = k_cache;
  a.v = v_cache;
  a.lengths = c.lengths = lengths;
  a.scale_log2 = c.scale_log2 = scale * 1.4426950408889634f;
  a.out = out;
  c.lse = a.lse = static_cast<float*>(workspace);
  c.part = a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + lse);
  c.scores = scores;
  if (int rc = ar_launch(fn, a, grid, as_stream(stream))) return rc;
  hipLaunchKernelGGL(attn_colsum_kernel, dim3(unsigned(cgrid)), dim3(256), 0, as_stream(stream), c);
  if (int rc = hip_status(fn)) return rc;
  hipLaunchKernelGGL(attn_colsum_add_kernel, dim3(unsigned(int64_t(B) * Hkv * c.nkt * (CS_KEYS / 64))),
                     dim3(256), 0, as_stream(stream), c);
  return hip_status(fn);
}
