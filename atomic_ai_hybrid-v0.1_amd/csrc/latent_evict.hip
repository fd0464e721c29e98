// Eviction from a paged cache by accumulated attention weight, for gfx950.
//
//   kept_b = the first `sinks` tokens, the `recent` newest, and of the rest the largest
//            weights (equal ones: the lowest rows), `keep` in all
//   row j < keep that was not kept  <-  the kept row >= keep of the same rank
//
// Selecting is integer work on 8 bytes a token and bound by latency; what moves are the
// kept rows past `keep` only, bound by their bytes.  So one workgroup a sequence selects
// and moves weights and order, and the rows are moved by a launch over the whole card.
#include "latent.hpp"

namespace ah {

struct EvictDims {
  int B, page, pages, table, width, keep, sinks, recent;
  int pieces;  // 16-byte pieces of a cache row
  int64_t ws, os, wos, oos;  // strides of weights, order and where the new ones go
};

// A weight as a number whose order is the float's: -0 as 0, a NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);
  return u >> 31 ? ~u : u | 0x80000000u;
}
constexpr uint32_t kSafe = 0xffffffffu;  // above every number's key

// The lanes below this one whose bit is set.
__device__ __forceinline__ int lanes_below(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;
constexpr int kDigit = 11, kBins = 1 << kDigit;  // 32 bits as 11, 11 and 10
constexpr int kEvictKeys = 1 << 15;              // keys that LDS holds (128 KB)

// Exclusive sum over the workgroup's waves; every thread of a wave gives the same x.
// `tmp` is not read any more when the call returns.
__device__ __forceinline__ int waves_below(int x, int* tmp, int& all) {
  if (lane_id() == 0) tmp[wave_id()] = x;
  __syncthreads();
  int below = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    if (w < wave_id()) below += tmp[w];
    sum += tmp[w];
  }
  __syncthreads();
  all = sum;
  return below;
}

// One sequence.  Its rows are divided over the waves in runs, so that ranks in the order of the
// rows are a wave's own count and the counts of the waves before it.  `keys` [width] a
// sequence hold what LDS has no room for (LDS = false), `movers` [keep] the kept rows
// past the budget.
template <bool LDS>
__global__ __launch_bounds__(kEvictThreads) void evict_select(EvictDims d, const int32_t* kv_lens, const float* weights,
                                                              const int32_t* order, int32_t* lens_out, float* w_out,
                                                              int32_t* o_out, int32_t* __restrict__ source,
                                                              uint32_t* __restrict__ key_space,
                                                              int32_t* __restrict__ mover_space) {
  __shared__ uint32_t skeys[LDS ? kEvictKeys : 1];
  __shared__ int hist[kBins];
  __shared__ int tmp[kEvictWaves], red[3], found[2];
  const int b = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  const int len = (int)min((int64_t)max(kv_lens[b], 0), (int64_t)d.table * d.page), left = min(len, d.keep);
  const float* w = weights + b * d.ws;
  const int32_t* o = order + b * d.os;
  uint32_t* keys = LDS ? skeys : key_space + (int64_t)b * d.width;
  int32_t* movers = mover_space + (int64_t)b * d.keep;
  source += (int64_t)b * d.keep;
  w_out += b * d.wos;
  o_out += b * d.oos;

  // what no eviction has seen: from row `first` to row `last`; the largest order of the others
  if (tid < 3) red[tid] = tid ? -1 : INT32_MAX;
  __syncthreads();
  int first = INT32_MAX, last = -1, top = -1;
  for (int j = tid; j < len; j += kEvictThreads) {
    const int x = o[j];
    if (x < 0) {
      first = min(first, j);
      last = max(last, j);
    } else {
      top = max(top, x);
    }
  }
#pragma unroll
  for (int k = 32; k; k >>= 1) {
    first = min(first, __shfl_xor(first, k));
    last = max(last, __shfl_xor(last, k));
    top = max(top, __shfl_xor(top, k));
  }
  if (lane == 0) {
    atomicMin(&red[0], first);
    atomicMax(&red[1], last);
    atomicMax(&red[2], top);
  }
  __syncthreads();
  first = red[0];
  last = red[1];
  top = red[2];
  const int64_t newest = last < 0 ? top : (int64_t)top + 1 + last - first;
  auto age = [&](int j) {  // the order of row j's token
    const int x = o[j];
    return x >= 0 ? (int64_t)x : (int64_t)top + 1 + j - first;
  };

  if (len > d.keep) {
    const int run = ((len + kEvictThreads - 1) / kEvictThreads) * 64;  // rows of a wave, whole lanes
    const int j0 = min(len, wave_id() * run), j1 = min(len, j0 + run);
    // f(row, here): all lanes of the wave together
    auto rows = [&](auto f) {
      for (int j = j0 + lane; j - lane < j1; j += 64) f(j, j < j1);
    };
    // the keep-th largest key, digit by digit from the top: `low` its digits so far, `need`
    // how many keys that begin with them are kept
    uint32_t low = 0;
    int need = d.keep, many = 0, shift = 32;
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? kDigit : 32 - 2 * kDigit;
      for (int i = tid; i < kBins; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      rows([&](int j, bool here) {
        if (!here) return;
        uint32_t k;
        if (pass == 0) {
          const int64_t a = age(j);
          k = a < d.sinks || a > newest - d.recent ? kSafe : weight_key(w[j]);
          keys[j] = k;
        } else {
          k = keys[j];
          if ((k >> shift) != (low >> shift)) return;
        }
        atomicAdd(&hist[(k >> (shift - bits)) & ((1 << bits) - 1)], 1);
      });
      __syncthreads();
      // keys in the bins above each bin: two bins a thread, from the top
      const int hi = kBins - 1 - 2 * tid, c0 = hist[hi], c1 = hist[hi - 1];
      int sum = c0 + c1;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const int y = __shfl_up(sum, k);
        if (lane >= k) sum += y;
      }
      int all;
      const int above = waves_below(__shfl(sum, 63), tmp, all) + sum - c0 - c1;
      if (above < need && need <= above + c0) {
        found[0] = hi;
        found[1] = above;
      } else if (above + c0 < need && need <= above + c0 + c1) {
        found[0] = hi - 1;
        found[1] = above + c0;
      }
      __syncthreads();
      shift -= bits;
      low |= (uint32_t)found[0] << shift;
      need -= found[1];
      many = hist[found[0]];
      __syncthreads();
      if (many == need) break;  // all that begin with `low` are kept: the last digits do not matter
    }
    // `need` of the keys that begin with `low` are kept, the lowest rows first
    int equal = 0, all;
    if (many != need) {
      rows([&](int j, bool here) { equal += __popcll(__ballot(here && keys[j] == low)); });
      equal = waves_below(equal, tmp, all);
    }
    auto kept = [&](int j, bool here, int& eq) {
      const uint32_t k = here ? keys[j] : 0;
      if (many == need) return here && k >= low;
      const uint64_t same = __ballot(here && k == low);
      const bool stay = here && (k > low || (k == low && eq + lanes_below(same) < need));
      eq += __popcll(same);
      return stay;
    };
    int eq = equal, holes = 0, moving = 0;
    rows([&](int j, bool here) {
      const bool stay = kept(j, here, eq);
      holes += __popcll(__ballot(here && !stay && j < d.keep));
      moving += __popcll(__ballot(stay && j >= d.keep));
    });
    holes = waves_below(holes, tmp, all);
    moving = waves_below(moving, tmp, all);
    eq = equal;
    rows([&](int j, bool here) {
      const bool stay = kept(j, here, eq);
      const uint64_t goes = __ballot(stay && j >= d.keep), free = __ballot(here && !stay && j < d.keep);
      if (stay && j >= d.keep) movers[moving + lanes_below(goes)] = j;
      if (here && j < d.keep) source[j] = stay ? j : ~(holes + lanes_below(free));  // a hole: its rank
      moving += __popcll(goes);
      holes += __popcll(free);
    });
    __threadfence_block();
    __syncthreads();
  }
  // the new state below the budget; then, when nothing past it is read any more, the rest
  for (int j = tid; j < left; j += kEvictThreads) {
    int from = j;
    if (len > d.keep) {
      from = source[j];
      if (from < 0) from = movers[~from];
    }
    const float x = w[from];
    const int a = (int)min(age(from), (int64_t)INT32_MAX);
    source[j] = from;
    w_out[j] = x;
    o_out[j] = a;
  }
  __syncthreads();
  for (int j = left + tid; j < d.width; j += kEvictThreads) {
    w_out[j] = 0.f;
    o_out[j] = -1;
  }
  for (int j = left + tid; j < d.keep; j += kEvictThreads) source[j] = -1;
  if (tid == 0) lens_out[b] = left;
}

// Cache rows: 64 rows of a sequence a workgroup, those of them that come from elsewhere.
constexpr int kMoveRows = 64;
__global__ __launch_bounds__(256) void evict_move(EvictDims d, const int32_t* __restrict__ table,
                                                  const int32_t* __restrict__ source, u32x4* cache) {
  __shared__ int64_t to[kMoveRows], from[kMoveRows];
  __shared__ int count;
  const int b = blockIdx.y, j = kMoveRows * blockIdx.x + threadIdx.x;
  auto place = [&](int r) {
    const int pg = r / d.page;
    const int64_t p = min(max(table[(int64_t)b * d.table + pg], 0), d.pages - 1);
    return (p * d.page + (r - pg * d.page)) * d.pieces;
  };
  if (threadIdx.x < kMoveRows) {
    const int src = j < d.keep ? source[(int64_t)b * d.keep + j] : -1;
    const bool go = src >= 0 && src != j;
    const uint64_t m = __ballot(go);
    if (go) {
      to[lanes_below(m)] = place(j);
      from[lanes_below(m)] = place(src);
    }
    if (threadIdx.x == 0) count = __popcll(m);
  }
  __syncthreads();
  const int n = count * d.pieces;
#pragma unroll 4
  for (int e = threadIdx.x; e < n; e += 256) {
    const int r = e / d.pieces, c = e - r * d.pieces;
    cache[to[r] + c] = cache[from[r] + c];
  }
}

static int evict_check(const atomic_latent_evict_args* a) {
  if (!a) return ATOMIC_ERR_NULL;
  if (a->dtype != ATOMIC_F32 && a->dtype != ATOMIC_BF16) return ATOMIC_ERR_DTYPE;
  if (a->batch < 1 || a->batch > 65535 || a->row < 16 || a->row > 576 || a->row % 8 || a->page < 1 || a->pages < 1 ||
      a->table_pages < 1 || (int64_t)a->table_pages * a->page > (1 << 30) ||
      a->width < (int64_t)a->table_pages * a->page || a->keep < 1 || a->keep > (1 << 30) || a->sinks < 0 || a->recent < 0 ||
      (int64_t)a->sinks + a->recent > a->keep || a->weights_stride < a->width || a->order_stride < a->width ||
      a->weights_out_stride < a->width || a->order_out_stride < a->width)
    return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}
// Rows that a sequence can have.
static int64_t evict_most(const atomic_latent_evict_args* a) { return (int64_t)a->table_pages * a->page; }

}  // namespace ah

using namespace ah;

extern "C" size_t atomic_latent_evict_workspace_size(const atomic_latent_evict_args* a) {
  if (evict_check(a) != ATOMIC_OK) return 0;
  const size_t keys = evict_most(a) > kEvictKeys ? (size_t)a->batch * a->width : 0;
  return (keys + (size_t)a->batch * a->keep) * 4;
}

extern "C" int atomic_latent_evict(const atomic_latent_evict_args* a, void* cache, const int32_t* page_table,
                                   const int32_t* kv_lens, const float* weights, const int32_t* order,
                                   int32_t* kv_lens_out, float* weights_out, int32_t* order_out, int32_t* source,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = evict_check(a)) return rc;
  if (!cache || !page_table || !kv_lens || !weights || !order || !kv_lens_out || !weights_out || !order_out || !source)
    return ATOMIC_ERR_NULL;
  if (!aligned16({cache})) return ATOMIC_ERR_SHAPE;
  const size_t bytes = atomic_latent_evict_workspace_size(a);
  if (!workspace || workspace_bytes < bytes || !aligned16({workspace})) return ATOMIC_ERR_WORKSPACE;
  ws_tag_clobber(workspace, bytes);
  const EvictDims d{a->batch, a->page, a->pages, a->table_pages, a->width, a->keep, a->sinks, a->recent,
                    a->row * (a->dtype == ATOMIC_BF16 ? 2 : 4) / 16, a->weights_stride, a->order_stride,
                    a->weights_out_stride, a->order_out_stride};
  const hipStream_t st = (hipStream_t)stream;
  Launch L{a->profile, st};
  int32_t* movers = (int32_t*)workspace;
  uint32_t* keys = (uint32_t*)workspace + (size_t)a->batch * a->keep;
  int rc = L("evict_select", [&] {
    if (evict_most(a) <= kEvictKeys)
      hipLaunchKernelGGL(evict_select<true>, dim3((unsigned)d.B), dim3(kEvictThreads), 0, st, d, kv_lens, weights,
                         order, kv_lens_out, weights_out, order_out, source, keys, movers);
    else
      hipLaunchKernelGGL(evict_select<false>, dim3((unsigned)d.B), dim3(kEvictThreads), 0, st, d, kv_lens, weights,
                         order, kv_lens_out, weights_out, order_out, source, keys, movers);
  });
  if (rc || evict_most(a) <= a->keep) return rc;
  return L("evict_move", [&] {
    hipLaunchKernelGGL(evict_move, dim3((unsigned)((d.keep + kMoveRows - 1) / kMoveRows), (unsigned)d.B), dim3(256),
                       0, st, d, page_table, source, (u32x4*)cache);
  });
}
