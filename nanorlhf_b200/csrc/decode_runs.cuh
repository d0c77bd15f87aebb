// What decode_flat.cu and decode_prefix.cuh share: the parameters of a decode call, and where parts lie.
#pragma once
#include "common.cuh"

namespace nrl {

constexpr int kPrefixRows = 64, kPrefixKeys = 64; // of a tile of query rows, of a step of the prefix

struct FlatParams {
  const __nv_bfloat16* q;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int *block_tables, *context_lens, *cu_groups, *shared;
  // what decode_plan finds
  int4* rows;                   // [S] first token that the row walks itself, pages of the rows in front (of one kv head), its own pages, its prefix's group + 1 (0: none);
                                // [S]: -, pages of all rows, pages a run, runs that have been taken
  int4* starts;                 // [runs] row, kv head, page of the row's own, -
  int4* groups;                 // [n_groups] steps of 64 tokens, of all heads and tiles, of the groups in front, the group's own (of a tile), its tokens that any of
                                // its rows sees, its query rows (of one kv head); [n_groups]: all steps, steps a run, -, -
  int4* prefix_starts;          // [prefix_runs] group, kv head x tiles + tile, step of the tile, -
  float *part_o, *part_ml;      // [runs + S Hkv, 8, D], [.., 8, 2]
  float* raw;                   // scores in log2 units [S, Hkv, G, 16 max_blocks] (null: none)
  float *prefix_o, *prefix_ml;  // [S Hq + 64 prefix_runs, D], [.., 2]: of run c, row i of all query rows (prefix_part_row) lies at i + 64 c
  __nv_bfloat16* out;
  const float* scores_in;
  float* scores_out;
  long q_stride_s, in_row, in_head, out_row, out_head;
  int n_groups, prefix_runs, blocks, S, max_blocks, Hq, Hkv, G, runs, least, max_tokens, chunk, wide, num_sms, near;
  int step_cost;                // of a step of a prefix, in pages of a row
  float scale_log2, decay;
};

NRL_DEVICE int flat_context(const FlatParams& p, int s) { return max(0, min(p.context_lens[s], p.max_blocks * 16)); }
NRL_DEVICE int prefix_tiles(int rows) { return (rows + kPrefixRows - 1) / kPrefixRows; }
// a query row among all: by group, kv head, sample and head
NRL_DEVICE long prefix_part_row(const FlatParams& p, int first, int h, int rows, int row) {
  return static_cast<long>(first) * p.G * p.Hkv + static_cast<long>(h) * rows + row;
}

}  // namespace nrl
