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
constexpr int kEvictList = 1 << 10;              // rows that move, as LDS holds them

// Exclusive sums of x and y over the workgroup's waves; every thread of a wave gives the same.
// `tmp` may be written again behind the caller's next barrier but one.
__device__ __forceinline__ void waves_below(int& x, int& y, int2* tmp) {
  if (lane_id() == 0) tmp[wave_id()] = make_int2(x, y);
  __syncthreads();
  x = y = 0;
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    const int2 z = tmp[w];
    x += w < wave_id() ? z.x : 0;
    y += w < wave_id() ? z.y : 0;
  }
}

// One sequence.  Its rows are divided over the waves in runs, so that ranks in the order of the
// rows are a wave's own count and the counts of the waves before it; a thread has eight rows in
// flight at a time.  `key_space` [width] a sequence holds the keys that LDS has no room for
// (LDS = false), `list_space` [keep] pairs of a hole and the kept row that goes there, past
// the first kEvictList of them.
//
// Bound by latency and, in a long table, by what one CU can read.
template <bool LDS>
__global__ __launch_bounds__(kEvictThreads) void evict_select(EvictDims d, const int32_t* kv_lens, const float* weights,
                                                              const int32_t* order, int32_t* lens_out, float* w_out,
                                                              int32_t* o_out, int32_t* __restrict__ source,
                                                              uint32_t* __restrict__ key_space,
                                                              int2* __restrict__ list_space) {
  __shared__ uint32_t skeys[LDS ? kEvictKeys : 1];
  __shared__ int hist[kBins];
  __shared__ int2 list[kEvictList];
  __shared__ int2 tmp[2][kEvictWaves];
  __shared__ int red[3], found[3];
  const int b = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  const int len = (int)min((int64_t)max(kv_lens[b], 0), (int64_t)d.table * d.page), left = min(len, d.keep);
  const float* w = weights + b * d.ws;
  const int32_t* o = order + b * d.os;
  uint32_t* keys = LDS ? skeys : key_space + (int64_t)b * d.width;
  int2* more = list_space + (int64_t)b * d.keep;
  source += (int64_t)b * d.keep;
  w_out += b * d.wos;
  o_out += b * d.oos;

  const int run = ((len + kEvictThreads - 1) / kEvictThreads) * 64;  // rows of a wave, whole lanes
  const int j0 = min(len, wave_id() * run), j1 = min(len, j0 + run);
  // f(i, j): eight times 64 rows of this wave, all lanes together; load(i, j) of them all before
  auto rows = [&](auto load, auto f) {
    for (int j = j0 + lane; j - lane < j1; j += 512) {
#pragma unroll
      for (int i = 0; i < 8; ++i) load(i, min(j + 64 * i, j1 - 1));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j - lane + 64 * i < j1) f(i, j + 64 * i, j + 64 * i < j1);
    }
  };

  // what no eviction has seen: from row `first` to row `last`; the largest order of the others
  if (tid < 3) red[tid] = tid ? -1 : INT32_MAX;
  for (int i = tid; i < kBins; i += kEvictThreads) hist[i] = 0;
  __syncthreads();
  int first = INT32_MAX, last = -1, top = -1, ages[8];
  rows([&](int i, int j) { ages[i] = o[j]; },
       [&](int i, int j, bool here) {
         const int x = ages[i];
         if (here && x < 0) {
           first = min(first, j);
           last = max(last, j);
         } else if (here) {
           top = max(top, x);
         }
       });
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
  // the order of row j's token where x stands there
  auto age = [&](int x, int j) { return x >= 0 ? (int64_t)x : (int64_t)top + 1 + j - first; };
  auto put = [&](int to, float x, int64_t a, int from) {
    source[to] = from;
    w_out[to] = x;
    o_out[to] = (int)min(a, (int64_t)INT32_MAX);
  };
  float ws[8];
  if (len <= d.keep) {
    rows(
        [&](int i, int j) {
          ages[i] = o[j];
          ws[i] = w[j];
        },
        [&](int i, int j, bool here) {
          if (here) put(j, ws[i], age(ages[i], j), j);
        });
  } else {
    // the keep-th largest key, digit by digit from the top: `low` its digits so far, `need`
    // how many of the `many` keys that begin with them are kept
    uint32_t low = 0, ks[8];
    int need = d.keep, many = 0, shift = 32;
    auto get = [&](int i, int j) { ks[i] = keys[j]; };
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? kDigit : 32 - 2 * kDigit;
      auto count = [&](uint32_t k) { atomicAdd(&hist[(k >> (shift - bits)) & ((1 << bits) - 1)], 1); };
      if (pass == 0) {
        rows(
            [&](int i, int j) {
              ages[i] = o[j];
              ws[i] = w[j];
            },
            [&](int i, int j, bool here) {
              const int64_t a = age(ages[i], j);
              const uint32_t k = a < d.sinks || a > newest - d.recent ? kSafe : weight_key(ws[i]);
              if (here) {
                keys[j] = k;
                count(k);
              }
            });
      } else {
        rows(get, [&](int i, int, bool here) {
          if (here && (ks[i] >> shift) == (low >> shift)) count(ks[i]);
        });
      }
      __syncthreads();
      // keys in the bins above each bin: two bins a thread, from the top
      const int hi = kBins - 1 - 2 * tid, c0 = hist[hi], c1 = hist[hi - 1];
      int sum = c0 + c1;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const int y = __shfl_up(sum, k);
        if (lane >= k) sum += y;
      }
      int above = __shfl(sum, 63), none = 0;
      waves_below(above, none, tmp[0]);
      above += sum - c0 - c1;
      if (above < need && need <= above + c0 + c1) {
        const bool lower = need > above + c0;
        found[0] = lower ? hi - 1 : hi;
        found[1] = lower ? above + c0 : above;
        found[2] = lower ? c1 : c0;
      }
      hist[hi] = hist[hi - 1] = 0;
      __syncthreads();
      shift -= bits;
      low |= (uint32_t)found[0] << shift;
      need -= found[1];
      many = found[2];
      if (many == need) break;  // all that begin with `low` are kept: the last digits do not matter
    }
    // `need` of the keys that begin with `low` are kept, the lowest rows first
    int equal = 0, none = 0;
    if (many != need) {
      rows(get, [&](int i, int, bool here) { equal += __popcll(__ballot(here && ks[i] == low)); });
      waves_below(equal, none, tmp[1]);
    }
    auto kept = [&](uint32_t k, bool here, int& eq) {
      if (many == need) return here && k >= low;
      const uint64_t same = __ballot(here && k == low);
      const bool stay = here && (k > low || (k == low && eq + lanes_below(same) < need));
      eq += __popcll(same);
      return stay;
    };
    int eq = equal, holes = 0, moving = 0;
    rows(get, [&](int i, int j, bool here) {
      const bool stay = kept(ks[i], here, eq);
      holes += __popcll(__ballot(here && !stay && j < d.keep));
      moving += __popcll(__ballot(stay && j >= d.keep));
    });
    waves_below(holes, moving, tmp[0]);
    eq = equal;
    rows(
        [&](int i, int j) {
          get(i, j);
          ages[i] = o[j];
          ws[i] = w[j];
        },
        [&](int i, int j, bool here) {
          const bool stay = kept(ks[i], here, eq), goes = stay && j >= d.keep, free = here && !stay && j < d.keep;
          const uint64_t gm = __ballot(goes), fm = __ballot(free);
          if (goes || free) {
            const int r = goes ? moving + lanes_below(gm) : holes + lanes_below(fm);
            int* at = (int*)(r < kEvictList ? list + r : more + r);
            at[goes] = j;
          } else if (stay) {
            put(j, ws[i], age(ages[i], j), j);
          }
          moving += __popcll(gm);
          holes += __popcll(fm);
        });
    // as many rows go as there are holes: the last wave's count
    if (wave_id() == kEvictWaves - 1 && lane == 0) found[0] = holes;
    __threadfence_block();
    __syncthreads();
    for (int r = tid; r < found[0]; r += kEvictThreads) {
      const int2 x = r < kEvictList ? list[r] : more[r];
      put(x.x, w[x.y], age(o[x.y], x.y), x.y);
    }
  }
  // past the length, when nothing there is read any more
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
  return (keys + 2 * (size_t)a->batch * a->keep) * 4;
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
  int2* list = (int2*)workspace;
  uint32_t* keys = (uint32_t*)(list + (size_t)a->batch * a->keep);
  int rc = L("evict_select", [&] {
    if (evict_most(a) <= kEvictKeys)
      hipLaunchKernelGGL(evict_select<true>, dim3((unsigned)d.B), dim3(kEvictThreads), 0, st, d, kv_lens, weights,
                         order, kv_lens_out, weights_out, order_out, source, keys, list);
    else
      hipLaunchKernelGGL(evict_select<false>, dim3((unsigned)d.B), dim3(kEvictThreads), 0, st, d, kv_lens, weights,
                         order, kv_lens_out, weights_out, order_out, source, keys, list);
  });
  if (rc || evict_most(a) <= a->keep) return rc;
  return L("evict_move", [&] {
    hipLaunchKernelGGL(evict_move, dim3((unsigned)((d.keep + kMoveRows - 1) / kMoveRows), (unsigned)d.B), dim3(256),
                       0, st, d, page_table, source, (u32x4*)cache);
  });
}
