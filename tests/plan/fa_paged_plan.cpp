// Host build of the paged calls' plans (libfa_mi355x.so's plan_paged) and of the
// arithmetic that their kernels share with them (csrc/fa_cache_kernels.h), for
// tests/test_paged_plan.py.
#include <stdint.h>

#include "fa_cache_kernels.h"

extern "C" {

// rows, slots, splits, chunk, conc, pieces, ws_rows, workspace_bytes
void paged_plan(int tokens, int batch, int kv_heads, int group, int head_dim, int max_q, int max_kv,
                int causal, int compute_units, int64_t* out) {
  const fa::PagedPlan p =
      fa::plan_paged(tokens, batch, kv_heads, group, head_dim, max_q, max_kv, causal != 0, compute_units);
  const fa::PagedGrid& g = p.grid;
  const int64_t v[8] = {g.rows, g.slots, g.splits, g.chunk, g.conc, g.pieces, (int64_t)g.ws_rows,
                        (int64_t)p.workspace_bytes};
  for (int i = 0; i < 8; ++i) out[i] = v[i];
}

// LastRound of a list of `found` tiles, its 64 lanes one after another: tiles
// listed, whole, rest, pieces.
void last_round(int found, int slots, int conc, int max_pieces, int max_kv, int* out) {
  const int count = fa::listed_tiles(found, slots), rest = count % conc;
  const float cost = fa::piece_cost(max_kv);
  int best = 1;
  float least = fa::cut_cost(rest, (rest + conc - 1) / conc, 1, max_pieces, cost);
  for (int q = 2; q <= 64; ++q) {
    const float c = fa::cut_cost(rest * q, (rest * q + conc - 1) / conc, q, max_pieces, cost);
    if (c < least) least = c, best = q;
  }
  out[0] = count, out[1] = count - rest, out[2] = rest, out[3] = best;
}

int64_t partial_tile(int kvh, int max_pieces, int tile, int pieces, int piece) {
  return fa::partial_tile(kvh, max_pieces, tile, pieces, piece);
}

}  // extern "C"
