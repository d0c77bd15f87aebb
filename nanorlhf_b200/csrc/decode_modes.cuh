// What the paged decode kernels do beside plain attention over a row's pages.
//   kDecodeTail    the row's group shares its first tokens, which another kernel (decode_prefix.cu) has attended to for all rows of the group: only the
//                  tokens behind them are walked, and the prefix's parts (maximum, sum, unnormalised result) are joined at the end
//   kDecodeScored  the scores of all tokens are left in scratch memory, for the weights that they come to once the row's maximum and sum are known
//                  (decode_scored.cu)
#pragma once
#include "common.cuh"

namespace nrl {

enum { kDecodePlain = 0, kDecodeTail = 1, kDecodeScored = 2 };

struct DecodeExtra {
  const int* cu_groups;          // [n_groups + 1] rows of the groups                     (tail)
  const int* shared;             // [n_groups] tokens that the rows of a group share
  int n_groups, prefix_parts;    // parts [0, prefix_parts) of a row are the prefix's
  float* raw;                    // [S, Hkv, G, raw_len] scores in log2 units             (scored)
  long raw_len;
};

// the group of a row, by a whole warp: cu is searched 32-fold; -1: none
NRL_DEVICE int group_of_row(const int* cu, int n, int row, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5, at = lo + lane * step;
    const uint32_t m = __ballot_sync(0xffffffffu, at < hi && cu[at] <= row);
    if (m == 0) return -1;
    lo += (__popc(m) - 1) * step;
    hi = min(hi, lo + step);
  }
  return n > 0 && cu[lo] <= row && row < cu[lo + 1] ? lo : -1;
}

struct DecodeFirst {
  int token;                     // the first that this row walks itself
  bool prefix;                   // its group has a prefix, and with it parts
};
template <int MODE>
NRL_DEVICE DecodeFirst decode_first(const DecodeExtra& x, int row, int ctx, int lane) {
  if (MODE != kDecodeTail) return {0, false};
  const int g = group_of_row(x.cu_groups, x.n_groups, row, lane);
  const int n = g >= 0 ? x.shared[g] : 0;
  return {max(0, min(n, ctx)), n > 0};
}

// parts of a row in all, and the place of one of its own
template <int MODE>
__host__ NRL_DEVICE int decode_parts(const DecodeExtra& x, int splits) { return MODE == kDecodeTail ? x.prefix_parts + splits : splits; }
template <int MODE>
NRL_DEVICE int decode_part(const DecodeExtra& x, int split) { return MODE == kDecodeTail ? x.prefix_parts + split : split; }

// A row's own part (M, L, acc: maximum, sum, element d of the result) takes up the prefix's parts where it is the only one; where a merge follows and there
// is no prefix, its parts are emptied.
template <int MODE>
NRL_DEVICE void decode_join_prefix(const DecodeExtra& x, DecodeFirst from, int splits, float* part_o, float* part_ml, long row, int split, int r, int d, float& M,
                                   float& L, float& acc) {
  if (MODE != kDecodeTail) return;
  const long base = row * decode_parts<MODE>(x, splits) * 8 + r;
  if (from.prefix && splits == 1) {
    float top = M;
    for (int s = 0; s < x.prefix_parts; ++s) top = fmaxf(top, part_ml[(base + s * 8) * 2]);
    const float own = M == -INFINITY ? 0.f : exp2f(M - top);
    L *= own;
    acc *= own;
    for (int s = 0; s < x.prefix_parts; ++s) {
      const float m = part_ml[(base + s * 8) * 2], c = m == -INFINITY ? 0.f : exp2f(m - top);
      L += part_ml[(base + s * 8) * 2 + 1] * c;
      acc += part_o[(base + s * 8) * 128 + d] * c;
    }
    M = top;
  } else if (!from.prefix && splits > 1 && split == 0) {
    for (int s = 0; s < x.prefix_parts; ++s) {
      part_o[(base + s * 8) * 128 + d] = 0.f;
      if (d == 0) {
        part_ml[(base + s * 8) * 2] = -INFINITY;
        part_ml[(base + s * 8) * 2 + 1] = 0.f;
      }
    }
  }
}

}  // namespace nrl
