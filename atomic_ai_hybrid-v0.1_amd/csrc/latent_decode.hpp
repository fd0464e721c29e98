// What the kernels of the absorbed form share: the sizes of a call and how the tokens of
// its sequences and prefixes are divided.
#pragma once
#include "latent.hpp"

namespace ah {

struct DecDims {
  int B, n, H, dn, dr, dv, dc, page, pages, table, rope, inter;
  int chunk, splits, groups;  // tokens a split (whole tiles), splits of the longest sequence, row groups
  float scale;
  int64_t qs[3];
  int share;         // latent_split: sequences whose rows read the same tokens (those of a prefix, or one)
  int slot0, slots;  // its first slot among a row's parts, and all of them
  int qn;            // rows that a query takes in q_lat: it, and where asked for what its rounding left out
  int part0;         // slots before the first whose part is fp32 (latent_prefix leaves its parts in its own way)
  // prefixes: sequences of each (0: there are none), tokens a split, slots, tokens their table holds, lengths
  int pre_share, pre_chunk, pre_splits, pre_most;
  const int32_t* pre_lens;
};
constexpr int kDecChunk = 1024, kDecPages = kDecChunk + 1;  // tokens of a split, pages that they can lie in
__device__ __forceinline__ int dec_len(const DecDims& d, const int32_t* kv_lens, int b) {
  return (int)min((int64_t)max(kv_lens[b], 0), (int64_t)d.table * d.page);
}
// Length of the prefix that sequence b's own tokens follow.
__device__ __forceinline__ int pre_len(const DecDims& d, int b) {
  return d.pre_share ? min(max(d.pre_lens[b / d.pre_share], 0), d.pre_most) : 0;
}
// The parts of sequence b's rows: those of the prefix's splits, then those of its own.
struct Parts {
  int front, all, skip;  // splits of the prefix, of both, slots to leave out between them
  __device__ __forceinline__ Parts(const DecDims& d, const int32_t* kv_lens, int b) {
    front = d.pre_share ? (pre_len(d, b) + d.pre_chunk - 1) / d.pre_chunk : 0;
    all = front + (d.splits ? (dec_len(d, kv_lens, b) + d.chunk - 1) / d.chunk : 0);
    skip = d.pre_splits - front;
  }
  __device__ __forceinline__ int slot(int s) const { return s < front ? s : s + skip; }
};

// Eight zeros: the source of the padding of a latent narrower than its tile.
static __device__ __attribute__((aligned(16))) const uint32_t lat_zeros[8] = {0, 0, 0, 0, 0, 0, 0, 0};

// latent_prefix: the prefixes' tokens against the rows of all sequences that follow them (bf16).
// Whether it takes the rows of `units` prefixes; divides their tokens for it, if so.
bool prefix_plan(DecDims& d, int units);
// Bytes of the parts that it leaves for the join.
size_t prefix_bytes(const DecDims& d, int units);
void launch_prefix(const DecDims& d, int units, hipStream_t st, const bf16* qa, const void* cache, const int32_t* table,
                   const int32_t* lens, const int32_t* own, int own_most, void* parts, float* stat);
// Joins them with those of the own tokens (`d`).  `shift`, unless NULL: a correction of each
// row's sum over the prefix (in its kernel's comment), in eight shares.
void launch_prefix_join(const DecDims& f, const DecDims& d, int units, hipStream_t st, const void* parts,
                        const float* part, const float* stat, const int32_t* kv_lens, float* olat, const bf16* qa,
                        float* shift);

}  // namespace ah
