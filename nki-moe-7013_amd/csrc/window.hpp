// What a query of a windowed attention sees, and the arguments that its entry points
// share.
#pragma once

#include "attn_tile.hpp"
#include "common.hpp"

#include <math.h>

namespace qmoe {

// r / G for 0 <= r < 2^32 / G, by a multiplication
__host__ __device__ __forceinline__ uint32_t ar_magic(uint32_t G) {
  return G == 1 ? 0u : uint32_t(((1ull << 32) + G - 1) / G);
}
__device__ __forceinline__ int ar_div(uint32_t r, uint32_t magic) { return int(magic ? __umulhi(r, magic) : r); }

constexpr int WIN_NONE = 1 << 30;  // no window: past every length

// Query s of row b stands at index p = ctx_len[b] - 1 + s and sees the entries
// e <= p with e > p - window or e < sink, and none from max_ctx on.
struct WinArgs {
  const int32_t* ctx_len;
  int S, S_max, max_ctx, window, sink;
};
struct WinRow {
  int low, end;  // sees [low, end) and [0, min(sink, end))
};
__device__ __forceinline__ WinRow win_row(const WinArgs& w, int b, int s) {
  const int n = min(max(w.ctx_len[b], -w.S), w.S_max) + s;  // p + 1
  return {max(n - w.window, 0), min(max(n, 0), w.max_ctx)};
}

// The run of keys that a tile of consecutive queries sees, whose first one's window
// begins at row `low` and whose last one sees rows below `end`: the first rows that
// stay, then the windows' (all of [low, end) is in one of them).  *n: keys of the run.
__device__ __forceinline__ Gap win_run(const WinArgs& w, int low, int end, int* n) {
  const int stay = min(w.sink, end);
  *n = low <= stay ? end : stay + max(end - low, 0);
  return {stay, max(low - stay, 0)};
}

// A cache in 4 bits: numbers [B][Hkv][S_max][64] and powers [B][Hkv][S_max][4].
struct Cache4 {
  const uint8_t *k, *ks, *v, *vs;
};

// ---------------------------------------------------------------------- host
// The calls of many rows, on the tiles of attn_rows.hip; cache: in 4 bits, instead of k
// and v.
int64_t attn_window_tiles_workspace(int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t max_ctx, int64_t window,
                                    int64_t sink);
int attn_window_tiles(const char* fn, const uint16_t* q, const uint16_t* k, const uint16_t* v, const Cache4* cache,
                      const int32_t* ctx_len, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t S_max,
                      int64_t max_ctx, int64_t window, int64_t sink, float scale, void* workspace,
                      int64_t workspace_bytes, uint16_t* out, hipStream_t stream);

inline WinArgs win_args(int64_t S, int64_t S_max, int64_t max_ctx, int64_t window, int64_t sink) {
  WinArgs w{};
  w.S = int(S);
  w.S_max = int(S_max);
  w.max_ctx = int(max_ctx);
  w.window = int(window == 0 ? WIN_NONE : std::min<int64_t>(window, WIN_NONE));
  w.sink = int(std::min<int64_t>(sink, WIN_NONE));
  return w;
}

inline int win_check(const char* fn, int64_t B, int64_t S, int64_t Hq, int64_t Hkv, int64_t D, int64_t S_max,
                     int64_t max_ctx, int64_t window, int64_t sink, float scale) {
  QMOE_REQUIRE(D == HD, "%s: head_dim must be 128 (D=%lld)", fn, (long long)D);
  QMOE_REQUIRE(Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Hq / Hkv <= 16 && Hkv < 4096,
               "%s: need Hq %% Hkv == 0, Hq / Hkv <= 16 and Hkv < 4096", fn);
  QMOE_REQUIRE(B >= 0 && B < 65536 && S >= 0 && S < (1ll << 22) && B * S * Hq < (1ll << 27),
               "%s: bad B/S (B * S * Hq must be below 2^27)", fn);
  // keys of a run are addressed with 32-bit byte offsets
  QMOE_REQUIRE(S_max > 0 && S_max <= (1ll << 22), "%s: S_max must be in [1, 2^22]", fn);
  QMOE_REQUIRE(max_ctx >= 0 && max_ctx <= S_max, "%s: need 0 <= max_ctx <= S_max", fn);
  QMOE_REQUIRE(window >= 0 && sink >= 0, "%s: window and sink must be >= 0", fn);
  QMOE_REQUIRE(scale > 0.0f && std::isfinite(scale), "%s: scale must be positive and finite", fn);
  return QMOE_OK;
}

// The rest of the checks, of B * S > 0 queries: the grid, `need` bytes of workspace,
// alignments and an output that is not q.
inline int win_operands(const char* fn, int64_t grid, int64_t need, const void* workspace, int64_t workspace_bytes,
                        const qmoe_bf16* q, const qmoe_bf16* out, int64_t heads) {
  QMOE_REQUIRE(grid < (1ll << 31), "%s: grid too large", fn);
  QMOE_REQUIRE(aligned16(q, static_cast<const uint8_t*>(workspace), out),
               "%s: operands must be 16-byte aligned", fn);
  const uintptr_t x = reinterpret_cast<uintptr_t>(q), y = reinterpret_cast<uintptr_t>(out);
  QMOE_REQUIRE((x < y ? y - x : x - y) >= uintptr_t(heads * AP_ROWB), "%s: out overlaps q", fn);
  QMOE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace of %lld bytes, need %lld", fn,
               (long long)workspace_bytes, (long long)need);
  return QMOE_OK;
}

}  // namespace qmoe
