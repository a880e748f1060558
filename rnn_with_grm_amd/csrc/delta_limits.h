// Sizes that the delta rule's launches do not take, for the C entry points and for the torch ops, which ask before they
// allocate anything.
#pragma once

#include <stdint.h>

namespace grmhip {

// The limit that a call passes, or null.  Sizes are at least zero; heads, value_dim and groups at least one, key_dim at most 128.
inline const char* delta_limit(int64_t batch, int64_t seq_len, int64_t heads, int64_t value_dim, int64_t groups, int64_t key_dim,
                               bool step) {
  const int64_t most = int64_t{1} << 21, grid = int64_t{1} << 24;
  if (seq_len > (1 << 30)) return "seq_len must be at most 2^30";
  // (One by one first: no product passes 63 bits.)
  if (heads > most || value_dim > most || groups > most || heads * value_dim > most || groups * key_dim > most)
    return "token strides and row widths must be at most 2^21 elements";
  // (A grid dimension has fewer than 2^32 threads, of which a workgroup of a walk and of the gradients has 512, of a token 256.)
  const int64_t seqs = heads * (batch < grid ? batch : grid), tiles = (value_dim + 63) / 64, chunks = (seq_len + 63) / 64;
  if (step) return seqs >= grid ? "batch * heads must be below 2^24" : nullptr;
  if (seqs >= grid || seqs * tiles >= grid / 2 || seqs * chunks >= grid / 2)
    return "batch * heads * ceil(value_dim / 64) and batch * heads * ceil(seq_len / 64) must be below 2^23";
  return nullptr;
}

}  // namespace grmhip
