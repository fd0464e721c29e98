// Eviction from a paged cache by accumulated attention weight, for gfx950.
//
//   kept_b = the first `sinks` tokens, the `recent` newest, and of the rest the largest
//            weights (equal ones: the lowest rows), `keep` in all
//   the k-th row below `keep` that was not kept  <-  the k-th kept row from `keep` on
//
// The keep-th largest weight is found digit by digit (11, 11 and 10 bits of a key whose
// order is the weight's) by counting how many keys have each digit; ranks in the order of
// the rows are sums of ballots.  All of it is integer work in a fixed result whatever the
// order of its atomics.  What moves are the kept rows past `keep` only.
//
// A table of up to 8192 tokens is selected from by one workgroup a sequence, its keys in
// registers (32 sequences of 8192: 13.6 us, in the other way 30); a longer one by many (one
// CU takes in about 10 bytes a clock of what is not in its cache: 131072 tokens took 200 us,
// in six launches 27), with a launch between the steps that need each other's sums.
#include "latent.hpp"

namespace ah {

struct EvictDims {
  int B, page, pages, table, width, keep, sinks, recent;
  int pieces;  // 16-byte pieces of a cache row
  int most;    // rows that a sequence can have
  int moves;   // and how many of them can move
  int fused;   // whether evict_small moves the cache rows itself
  int64_t ws, os, wos, oos;  // strides of weights, order and where the new ones go
};
struct EvictIn {
  const int32_t* lens;
  const float* w;
  const int32_t* o;
};
struct EvictOut {
  int32_t* lens;
  float* w;
  int32_t *o, *source;
};
// A row that moves: from where, with what.
struct __attribute__((aligned(16))) Mover {
  int from;
  float w;
  int order, to;
};

// A weight as a number whose order is the float's: -0 as 0, a NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);
  return u >> 31 ? ~u : u | 0x80000000u;
}
constexpr uint32_t kSafe = 0xffffffffu;  // above every number's key
constexpr int kDigit = 11, kBins = 1 << kDigit;
constexpr int kRows = 8;  // rows of a thread: 64 of a wave each

__device__ __forceinline__ int lanes_below(uint64_t mask) {  // the lanes below this one whose bit is set
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}
// Inclusive sum over a wave's lanes.
__device__ __forceinline__ int lanes_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}
// Largest of a wave's lanes (of numbers from -1 on).
__device__ __forceinline__ int lanes_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(-1, x, 0x111, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(-1, x, 0x112, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(-1, x, 0x114, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(-1, x, 0x118, 0xF, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(-1, x, 0x142, 0xA, 0xF, false));
  x = max(x, __builtin_amdgcn_update_dpp(-1, x, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(x, 63);
}

__device__ __forceinline__ int evict_len(const EvictDims& d, const int32_t* lens, int b) {
  return min(max(lens[b], 0), d.most);
}

// What no eviction has seen: from row `first` to row `last`; the largest order of the others.
struct Ages {
  int first, last, top;
  static __device__ __forceinline__ Ages none() { return Ages{INT32_MAX, -1, -1}; }
  __device__ __forceinline__ void add(int j, int x, bool here) {  // all lanes of a wave, rows in a run
    const uint64_t fresh = __ballot(here && x < 0);
    if (fresh) {
      const int j0 = __builtin_amdgcn_readfirstlane(j);
      first = min(first, j0 + (int)__builtin_ctzll(fresh));
      last = max(last, j0 + 63 - (int)__builtin_clzll(fresh));
    }
    top = max(top, here ? x : -1);
  }
  __device__ __forceinline__ void add(const Ages& x) {
    first = min(first, x.first);
    last = max(last, x.last);
    top = max(top, x.top);
  }
  // the order of row j's token where x stands there
  __device__ __forceinline__ int64_t of(int x, int j) const { return x >= 0 ? (int64_t)x : (int64_t)top + 1 + j - first; }
  __device__ __forceinline__ uint32_t key(const EvictDims& d, int x, int j, float w) const {
    const int64_t newest = last < 0 ? top : (int64_t)top + 1 + last - first, a = of(x, j);
    return a < d.sinks || a > newest - d.recent ? kSafe : weight_key(w);
  }
  __device__ __forceinline__ int put(int x, int j) const { return (int)min(of(x, j), (int64_t)INT32_MAX); }
};

// The keep-th largest key, as far as its digits are known: `low`, those so far, `need`
// how many of the `many` keys that begin with them are kept.  `hist` counts the next digit;
// the call clears it where it is LDS, and ends with a barrier.
struct Digits {
  uint32_t low = 0;
  int need, many = -1, shift = 32;
  __device__ __forceinline__ bool done() const { return many == need || shift == 0; }
  __device__ __forceinline__ int bits() const { return shift > 10 ? kDigit : 10; }
  __device__ __forceinline__ bool begins(uint32_t k) const { return shift == 32 || (k >> shift) == (low >> shift); }
  __device__ __forceinline__ int bin(uint32_t k) const { return (k >> (shift - bits())) & ((1 << bits()) - 1); }
  template <int NT, bool LDS>
  __device__ __forceinline__ void next(int* hist, int* tmp, int* found) {
    constexpr int NB = kBins / NT, NW = NT / 64;
    const int lane = lane_id(), hi = kBins - 1 - NB * (int)threadIdx.x;  // this thread's bins, from the top
    int c[NB], sum = 0;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      c[i] = hist[hi - i];
      sum += c[i];
    }
    int above = lanes_sum(sum);
    if (lane == 63) tmp[wave_id()] = above;
    above -= sum;
    if constexpr (LDS) {
#pragma unroll
      for (int i = 0; i < NB; ++i) hist[hi - i] = 0;
    }
    __syncthreads();
    const int t = lanes_sum(lane < NW ? tmp[lane] : 0);
    if (wave_id()) above += __builtin_amdgcn_readlane(t, max(wave_id() - 1, 0));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      if (above < need && need <= above + c[i]) {
        found[0] = hi - i;
        found[1] = above;
        found[2] = c[i];
      }
      above += c[i];
    }
    __syncthreads();
    shift -= bits();
    low |= (uint32_t)found[0] << shift;
    need -= found[1];
    many = found[2];
  }
  // Whether key k is kept; `eq` counts the equal ones before, by the order of the rows.
  __device__ __forceinline__ bool kept(uint32_t k, bool here, int& eq) const {
    if (many == need) return here && k >= low;  // all that begin with `low`
    const uint64_t same = __ballot(here && k == low);
    const bool stay = here && (k > low || (k == low && eq + lanes_below(same) < need));
    eq += __popcll(same);
    return stay;
  }
};

// Exclusive sums of x and y over the workgroup's waves (every lane of a wave gives the same), and their totals.
template <int NT>
__device__ __forceinline__ void waves_below(int& x, int& y, int2* tmp, int2& all) {
  constexpr int NW = NT / 64;
  if (lane_id() == 0) tmp[wave_id()] = make_int2(x, y);
  __syncthreads();
  const int2 z = tmp[min(lane_id(), NW - 1)];
  const int sx = lanes_sum(lane_id() < NW ? z.x : 0), sy = lanes_sum(lane_id() < NW ? z.y : 0);
  all = make_int2(__builtin_amdgcn_readlane(sx, NW - 1), __builtin_amdgcn_readlane(sy, NW - 1));
  x = __builtin_amdgcn_readlane(sx, wave_id()) - x;
  y = __builtin_amdgcn_readlane(sy, wave_id()) - y;
}

__device__ __forceinline__ int64_t cache_piece(const EvictDims& d, const int32_t* table, int b, int r) {
  const int pg = r / d.page;
  const int64_t p = min(max(table[(int64_t)b * d.table + pg], 0), d.pages - 1);
  return (p * d.page + (r - pg * d.page)) * d.pieces;
}

// ------------------------------------------------------------------ short tables
// One sequence, its rows in runs of a wave each: bound by the latency of its steps (10 us with
// 2048 rows, 14 with 8192).  The loads of all rows are sent before the length is known.  Where few rows can move (`fused`: the step of a full cache) it
// moves them too, which saves a launch; else it leaves them in `movers` [moves] and `count`.
template <int NT>
__global__ __launch_bounds__(NT) void evict_small(EvictDims d, EvictIn in, EvictOut out,
                                                  const int32_t* __restrict__ table, u32x4* cache,
                                                  Mover* __restrict__ movers, int32_t* __restrict__ count) {
  constexpr int NW = NT / 64, KEEP = kRows * NT / 2;  // (no more rows move than half of them)
  __shared__ int hist[kBins];
  __shared__ int holes_at[KEEP];
  __shared__ Mover mv[KEEP];
  __shared__ int2 tmp2[2][NW];
  __shared__ int tmp[NW], found[3];
  __shared__ Ages sa[NW];
  const int b = blockIdx.x, tid = threadIdx.x, lane = lane_id();
  const float* w = in.w + b * d.ws;
  const int32_t* o = in.o + b * d.os;
  const int per = (d.most + NT - 1) / NT;  // rows of a thread
  const int j0 = wave_id() * 64 * per + lane;
  int x[kRows];
  float v[kRows];
  uint32_t k[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (i < per) {
      const int j = min(j0 + 64 * i, d.most - 1);
      x[i] = o[j];
      v[i] = w[j];
    }
  const int len = evict_len(d, in.lens, b), left = min(len, d.keep);
  for (int i = tid; i < kBins; i += NT) hist[i] = 0;
  Ages ages = Ages::none();
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (i < per) ages.add(j0 + 64 * i, x[i], j0 + 64 * i < len);
  ages.top = lanes_max(ages.top);
  if (lane == 0) sa[wave_id()] = ages;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NW; ++i) ages.add(sa[i]);
  int* source = out.source + (int64_t)b * d.keep;
  float* w_out = out.w + b * d.wos;
  int32_t* o_out = out.o + b * d.oos;
  int n = 0;
  if (len <= d.keep) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int j = j0 + 64 * i;
      if (i < per && j < len) {
        source[j] = j;
        w_out[j] = v[i];
        o_out[j] = ages.put(x[i], j);
      }
    }
  } else {
    Digits g;
    g.need = d.keep;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i < per) {
        const int j = j0 + 64 * i;
        k[i] = ages.key(d, x[i], j, v[i]);
      }
    do {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (i < per && j0 + 64 * i < len && g.begins(k[i])) atomicAdd(&hist[g.bin(k[i])], 1);
      __syncthreads();
      g.next<NT, true>(hist, tmp, found);
    } while (!g.done());
    int equal = 0, none = 0;
    int2 all;
    if (g.many != g.need) {
#pragma unroll
      for (int i = 0; i < kRows; ++i)
        if (i < per) equal += __popcll(__ballot(j0 + 64 * i < len && k[i] == g.low));
      waves_below<NT>(equal, none, tmp2[0], all);
    }
    uint32_t stays = 0;
    int holes = 0, moving = 0;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i < per) {
        const int j = j0 + 64 * i;
        const bool stay = g.kept(k[i], j < len, equal);
        stays |= (uint32_t)stay << i;
        holes += __popcll(__ballot(j < d.keep && !stay));
        moving += __popcll(__ballot(j >= d.keep && stay));
      }
    waves_below<NT>(holes, moving, tmp2[1], all);
    n = all.x;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i < per) {
        const int j = j0 + 64 * i;
        const bool stay = stays >> i & 1, goes = j >= d.keep && stay, free = j < d.keep && !stay;
        const uint64_t gm = __ballot(goes), fm = __ballot(free);
        if (goes) mv[moving + lanes_below(gm)] = Mover{j, v[i], ages.put(x[i], j), 0};
        if (free) holes_at[holes + lanes_below(fm)] = j;
        if (j < d.keep && stay) {
          source[j] = j;
          w_out[j] = v[i];
          o_out[j] = ages.put(x[i], j);
        }
        moving += __popcll(gm);
        holes += __popcll(fm);
      }
    __syncthreads();
    for (int r = tid; r < n; r += NT) {
      Mover m = mv[r];
      m.to = holes_at[r];
      source[m.to] = m.from;
      w_out[m.to] = m.w;
      o_out[m.to] = m.order;
      if (!d.fused) movers[(int64_t)b * d.moves + r] = m;
    }
  }
  // past the length (every row has been read; a state may end within a step of 2^31)
  for (int64_t j = left + tid; j < d.width; j += NT) {
    w_out[j] = 0.f;
    o_out[j] = -1;
  }
  for (int j = left + tid; j < d.keep; j += NT) source[j] = -1;
  if (tid == 0) {
    out.lens[b] = left;
    if (!d.fused && d.moves) count[b] = n;
  }
  if (d.fused) {  // (at most kFused rows)
    for (int e = tid; e < n * d.pieces; e += NT) {
      const int r = e / d.pieces, c = e - r * d.pieces;
      cache[cache_piece(d, table, b, holes_at[r]) + c] = cache[cache_piece(d, table, b, mv[r].from) + c];
    }
  }
}
// Rows that evict_small moves itself.  (64 sequences of 2048 tokens and more, us: 9.8 of 1 row each, 22 of 128, 34 of
// 256; with evict_move 9.8 + 4, 9.7 + 8.7 and 9.4 + 9.6, and a launch's gap.)
constexpr int kFused = 96;

// ------------------------------------------------------------------ long tables
// 2048 rows a workgroup; those below `keep` and those from it on are divided apart.  Each
// launch leaves its counts in a sequence's share of the workspace for the next:
//   evict_ages    first / last / top of each chunk; clears the histograms
//   evict_digit   (three times) the keys, and how many have each digit
//   evict_count   kept for certain, and equal to the last one, of each chunk
//   evict_emit    the kept rows' new state; the rows that move and where to, by rank
constexpr int kChunk = 256 * kRows;
struct EvictLong {
  int chunks, below;  // of a sequence, and those of them below `keep`
  Ages* ages;         // [B, chunks]
  int* hist;          // [B, 3, kBins]
  int2* counts;       // [B, chunks]
  uint32_t* keys;     // [B, most]
  int32_t* left;      // [B], the new lengths
};
struct Chunk {
  int b, c, j0, end, len;
  __device__ __forceinline__ Chunk(const EvictDims& d, const EvictLong& x, const int32_t* lens) {
    b = blockIdx.y;
    c = blockIdx.x;
    len = evict_len(d, lens, b);
    const int from = c < x.below ? c * kChunk : d.keep + (c - x.below) * kChunk;
    end = min(len, c < x.below ? min(d.keep, from + kChunk) : from + kChunk);
    j0 = from + wave_id() * 64 * kRows + lane_id();
  }
};
__device__ __forceinline__ Ages all_ages(const EvictLong& x, int b, Ages* sa) {
  Ages a = Ages::none();
  for (int i = threadIdx.x; i < x.chunks; i += 256) a.add(x.ages[(int64_t)b * x.chunks + i]);
  a.first = INT32_MAX - 1 - lanes_max(INT32_MAX - 1 - min(a.first, INT32_MAX - 1));
  a.last = lanes_max(a.last);
  a.top = lanes_max(a.top);
  if (lane_id() == 0) sa[wave_id()] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) a.add(sa[i]);
  __syncthreads();
  return a;
}
__global__ __launch_bounds__(256) void evict_ages(EvictDims d, EvictIn in, EvictLong x) {
  __shared__ Ages sa[4];
  const Chunk c(d, x, in.lens);
  const int32_t* o = in.o + c.b * d.os;
  int y[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) y[i] = o[min(c.j0 + 64 * i, d.most - 1)];
  Ages a = Ages::none();
#pragma unroll
  for (int i = 0; i < kRows; ++i) a.add(c.j0 + 64 * i, y[i], c.j0 + 64 * i < c.end);
  a.top = lanes_max(a.top);
  if (lane_id() == 0) sa[wave_id()] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 4; ++i) a.add(sa[i]);
    x.ages[(int64_t)c.b * x.chunks + c.c] = a;
  }
  for (int i = c.c * 256 + threadIdx.x; i < 3 * kBins; i += 256 * x.chunks) x.hist[(int64_t)c.b * 3 * kBins + i] = 0;
}
// The digits known before pass `passes`.
__device__ __forceinline__ Digits all_digits(const EvictDims& d, const EvictLong& x, int b, int passes, int* tmp,
                                             int* found) {
  Digits g;
  g.need = d.keep;
  for (int p = 0; p < passes && !g.done(); ++p) g.next<256, false>(x.hist + ((int64_t)b * 3 + p) * kBins, tmp, found);
  return g;
}
__global__ __launch_bounds__(256) void evict_digit(EvictDims d, EvictIn in, EvictLong x, int pass) {
  __shared__ int hist[kBins], tmp[4], found[3];
  __shared__ Ages sa[4];
  const Chunk c(d, x, in.lens);
  if (c.len <= d.keep) return;
  uint32_t* keys = x.keys + (int64_t)c.b * d.most;
  uint32_t k[kRows];
  for (int i = threadIdx.x; i < kBins; i += 256) hist[i] = 0;
  Digits g;
  if (pass == 0) {
    const float* w = in.w + c.b * d.ws;
    const int32_t* o = in.o + c.b * d.os;
    int y[kRows];
    float v[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int j = min(c.j0 + 64 * i, d.most - 1);
      y[i] = o[j];
      v[i] = w[j];
    }
    const Ages a = all_ages(x, c.b, sa);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int j = c.j0 + 64 * i;
      k[i] = a.key(d, y[i], j, v[i]);
      if (j < c.end) keys[j] = k[i];
    }
    g.need = d.keep;
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i) k[i] = keys[min(c.j0 + 64 * i, c.len - 1)];
    g = all_digits(d, x, c.b, pass, tmp, found);
    if (g.done()) return;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    if (c.j0 + 64 * i < c.end && g.begins(k[i])) atomicAdd(&hist[g.bin(k[i])], 1);
  __syncthreads();
  int* to = x.hist + ((int64_t)c.b * 3 + pass) * kBins;
  for (int i = threadIdx.x; i < kBins; i += 256)
    if (hist[i]) atomicAdd(to + i, hist[i]);
}
__global__ __launch_bounds__(256) void evict_count(EvictDims d, EvictIn in, EvictLong x) {
  __shared__ int tmp[4], found[3];
  __shared__ int2 tmp2[4];
  const Chunk c(d, x, in.lens);
  if (c.len <= d.keep) return;
  const uint32_t* keys = x.keys + (int64_t)c.b * d.most;
  uint32_t k[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) k[i] = keys[min(c.j0 + 64 * i, c.len - 1)];
  const Digits g = all_digits(d, x, c.b, 3, tmp, found);
  int sure = 0, equal = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const bool here = c.j0 + 64 * i < c.end, all = g.many == g.need;
    sure += __popcll(__ballot(here && (all ? k[i] >= g.low : k[i] > g.low)));
    equal += __popcll(__ballot(here && !all && k[i] == g.low));
  }
  int2 all;
  waves_below<256>(sure, equal, tmp2, all);
  if (threadIdx.x == 0) x.counts[(int64_t)c.b * x.chunks + c.c] = all;
}
__global__ __launch_bounds__(256) void evict_emit(EvictDims d, EvictIn in, EvictLong x, EvictOut out,
                                                  Mover* __restrict__ movers, int32_t* __restrict__ count) {
  __shared__ int tmp[4], found[3];
  __shared__ int2 tmp2[3][4];
  __shared__ Ages sa[4];
  const Chunk c(d, x, in.lens);
  if (c.c == 0 && threadIdx.x == 0) x.left[c.b] = min(c.len, d.keep);
  const float* w = in.w + c.b * d.ws;
  const int32_t* o = in.o + c.b * d.os;
  int y[kRows];
  float v[kRows];
  uint32_t k[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int j = min(c.j0 + 64 * i, d.most - 1);
    y[i] = o[j];
    v[i] = w[j];
  }
  const Ages a = all_ages(x, c.b, sa);
  int* source = out.source + (int64_t)c.b * d.keep;
  float* w_out = out.w + c.b * d.wos;
  int32_t* o_out = out.o + c.b * d.oos;
  auto put = [&](int i, int j) {
    source[j] = j;
    w_out[j] = v[i];
    o_out[j] = a.put(y[i], j);
  };
  if (c.len <= d.keep) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (c.j0 + 64 * i < c.end) put(i, c.j0 + 64 * i);
    if (c.c == 0 && threadIdx.x == 0) count[c.b] = 0;
    return;
  }
  const uint32_t* keys = x.keys + (int64_t)c.b * d.most;
#pragma unroll
  for (int i = 0; i < kRows; ++i) k[i] = keys[min(c.j0 + 64 * i, c.len - 1)];
  const Digits g = all_digits(d, x, c.b, 3, tmp, found);
  // equal keys, holes and moving rows in the chunks before; all of them
  const bool low = c.c < x.below;
  int eq = 0, before = 0, sure = 0, equal = 0;  // (a sum of equals by all lanes, of the rest below)
  for (int i = threadIdx.x; i < x.chunks; i += 256) {
    const int2 n = x.counts[(int64_t)c.b * x.chunks + i];
    if (i < c.c) eq += n.y;
    if (low ? i < c.c : i >= x.below && i < c.c) {
      sure += n.x;
      equal += n.y;
    }
    if (i < x.below) before += n.y;
  }
  int2 s0, s1;
  eq = __builtin_amdgcn_readlane(lanes_sum(eq), 63);
  before = __builtin_amdgcn_readlane(lanes_sum(before), 63);
  sure = __builtin_amdgcn_readlane(lanes_sum(sure), 63);
  equal = __builtin_amdgcn_readlane(lanes_sum(equal), 63);
  waves_below<256>(eq, before, tmp2[0], s0);
  waves_below<256>(sure, equal, tmp2[1], s1);
  // of the equal keys the first `need` in the order of the rows are kept
  const int first = low ? 0 : s0.y;  // equal keys before this side of `keep`
  const int kept = s1.x + min(max(g.need - first, 0), s1.y);
  const int rows = c.c * kChunk;  // (below `keep` only full chunks lie before)
  int rank = low ? rows - kept : kept, here_eq = 0, none = 0;
  eq = s0.x;
#pragma unroll
  for (int i = 0; i < kRows; ++i) here_eq += __popcll(__ballot(c.j0 + 64 * i < c.end && k[i] == g.low));
  int2 all;
  waves_below<256>(here_eq, none, tmp2[2], all);
  eq += here_eq;
  uint32_t stays = 0;
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int j = c.j0 + 64 * i;
    const bool stay = g.kept(k[i], j < c.end, eq);
    stays |= (uint32_t)stay << i;
    mine += __popcll(__ballot(j < c.end && stay != low));  // holes below `keep`, moving rows from it on
  }
  none = 0;
  waves_below<256>(mine, none, tmp2[0], all);
  if (c.c == x.below - 1 && threadIdx.x == 0) count[c.b] = rank + all.x;
  rank += mine;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int j = c.j0 + 64 * i;
    const bool stay = stays >> i & 1, takes = j < c.end && stay != low;
    const uint64_t m = __ballot(takes);
    Mover* to = movers + (int64_t)c.b * d.moves + rank + lanes_below(m);
    if (takes && low) {
      to->to = j;
    } else if (takes) {
      to->from = j;
      to->w = v[i];
      to->order = a.put(y[i], j);
    } else if (stay) {
      put(i, j);
    }
    rank += __popcll(m);
  }
}

// Cache rows, 64 that move a workgroup: bound by their bytes, read and written in rows that lie
// scattered (32 sequences of 4100 to 8192 tokens to 2048: 25 us for 107 MB, 4.2 TB/s).  With STATE the moved rows' weights and order as well, and what lies past the length.
constexpr int kMoveRows = 64;
template <bool STATE>
__global__ __launch_bounds__(256) void evict_move(EvictDims d, const int32_t* __restrict__ table,
                                                  const Mover* __restrict__ movers, const int32_t* __restrict__ count,
                                                  EvictOut out, const int32_t* __restrict__ left_of, u32x4* cache) {
  __shared__ int64_t to[kMoveRows], from[kMoveRows];
  const int b = blockIdx.y, r0 = kMoveRows * blockIdx.x, n = min(count[b] - r0, kMoveRows);
  float* w_out = out.w + b * d.wos;
  int32_t* o_out = out.o + b * d.oos;
  int* source = out.source + (int64_t)b * d.keep;
  if constexpr (STATE) {
    const int left = left_of[b];
    const int64_t first = left + 256 * (int64_t)blockIdx.x + threadIdx.x, step = 256 * (int64_t)gridDim.x;
    for (int64_t j = first; j < d.width; j += step) {
      w_out[j] = 0.f;
      o_out[j] = -1;
    }
    for (int64_t j = first; j < d.keep; j += step) source[j] = -1;
    if (blockIdx.x == 0 && threadIdx.x == 0) out.lens[b] = left;
  }
  if (n <= 0) return;
  if ((int)threadIdx.x < n) {
    const Mover m = movers[(int64_t)b * d.moves + r0 + threadIdx.x];
    to[threadIdx.x] = cache_piece(d, table, b, m.to);
    from[threadIdx.x] = cache_piece(d, table, b, m.from);
    if constexpr (STATE) {
      source[m.to] = m.from;
      w_out[m.to] = m.w;
      o_out[m.to] = m.order;
    }
  }
  __syncthreads();
#pragma unroll 4
  for (int e = threadIdx.x; e < n * d.pieces; e += 256) {
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

// How a call goes: where its parts lie in the workspace, which kernels take it.
struct EvictPlan {
  EvictDims d;
  bool small;
  EvictLong x;
  size_t movers, count, left, ages, counts, hist, keys, all;
};
static EvictPlan evict_plan(const atomic_latent_evict_args* a) {
  EvictPlan p{};
  const int most = a->table_pages * a->page, over = most > a->keep ? most - a->keep : 0;
  p.d = EvictDims{a->batch, a->page, a->pages, a->table_pages, a->width, a->keep, a->sinks, a->recent,
                  a->row * (a->dtype == ATOMIC_BF16 ? 2 : 4) / 16, most, a->keep < over ? a->keep : over, 0,
                  a->weights_stride, a->order_stride, a->weights_out_stride, a->order_out_stride};
  p.small = most <= kRows * 1024;
  p.d.fused = p.small && p.d.moves <= kFused;
  p.x.below = ((a->keep < most ? a->keep : most) + kChunk - 1) / kChunk;
  p.x.chunks = p.x.below + (over + kChunk - 1) / kChunk;
  size_t at = 0;
  auto part = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t B = (size_t)a->batch, chunks = p.small ? 0 : B * p.x.chunks;
  p.movers = part(p.d.fused ? 0 : B * p.d.moves * sizeof(Mover));
  p.count = part(B * sizeof(int32_t));
  p.left = part(B * sizeof(int32_t));
  p.ages = part(chunks * sizeof(Ages));
  p.counts = part(chunks * sizeof(int2));
  p.hist = part(p.small ? 0 : B * 3 * kBins * sizeof(int));
  p.keys = part(p.small ? 0 : B * most * sizeof(uint32_t));
  p.all = at;
  return p;
}

}  // namespace ah

using namespace ah;

extern "C" size_t atomic_latent_evict_workspace_size(const atomic_latent_evict_args* a) {
  return evict_check(a) == ATOMIC_OK ? evict_plan(a).all : 0;
}

extern "C" int atomic_latent_evict(const atomic_latent_evict_args* a, void* cache, const int32_t* page_table,
                                   const int32_t* kv_lens, const float* weights, const int32_t* order,
                                   int32_t* kv_lens_out, float* weights_out, int32_t* order_out, int32_t* source,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = evict_check(a)) return rc;
  if (!cache || !page_table || !kv_lens || !weights || !order || !kv_lens_out || !weights_out || !order_out || !source)
    return ATOMIC_ERR_NULL;
  if (!aligned16({cache})) return ATOMIC_ERR_SHAPE;
  EvictPlan p = evict_plan(a);
  if (!workspace || workspace_bytes < p.all || !aligned16({workspace})) return ATOMIC_ERR_WORKSPACE;
  ws_tag_clobber(workspace, p.all);
  const EvictDims& d = p.d;
  const hipStream_t st = (hipStream_t)stream;
  Launch L{a->profile, st};
  char* ws = (char*)workspace;
  Mover* movers = (Mover*)(ws + p.movers);
  int32_t *count = (int32_t*)(ws + p.count), *left = (int32_t*)(ws + p.left);
  const EvictIn in{kv_lens, weights, order};
  const EvictOut out{kv_lens_out, weights_out, order_out, source};
  const dim3 moves((unsigned)((d.moves + kMoveRows - 1) / kMoveRows), (unsigned)d.B);
  if (p.small) {
    const int rc = L("evict_small", [&] {
      auto go = [&](auto nt) {
        hipLaunchKernelGGL((evict_small<decltype(nt)::value>), dim3((unsigned)d.B), dim3(decltype(nt)::value), 0, st, d,
                           in, out, page_table, (u32x4*)cache, movers, count);
      };
      if (d.most <= kRows * 256) go(IntC<256>());
      else if (d.most <= kRows * 512) go(IntC<512>());
      else go(IntC<1024>());
    });
    if (rc || d.fused) return rc;
    return L("evict_move", [&] {
      hipLaunchKernelGGL(evict_move<false>, moves, dim3(256), 0, st, d, page_table, movers, count, out, left,
                         (u32x4*)cache);
    });
  }
  EvictLong x = p.x;
  x.ages = (Ages*)(ws + p.ages);
  x.counts = (int2*)(ws + p.counts);
  x.hist = (int*)(ws + p.hist);
  x.keys = (uint32_t*)(ws + p.keys);
  x.left = left;
  const dim3 grid((unsigned)x.chunks, (unsigned)d.B);
  int rc = L("evict_ages", [&] { hipLaunchKernelGGL(evict_ages, grid, dim3(256), 0, st, d, in, x); });
  if (d.moves) {
    for (int pass = 0; pass < 3 && !rc; ++pass)
      rc = L("evict_digit", [&] { hipLaunchKernelGGL(evict_digit, grid, dim3(256), 0, st, d, in, x, pass); });
    if (!rc) rc = L("evict_count", [&] { hipLaunchKernelGGL(evict_count, grid, dim3(256), 0, st, d, in, x); });
  }
  if (!rc) rc = L("evict_emit", [&] { hipLaunchKernelGGL(evict_emit, grid, dim3(256), 0, st, d, in, x, out, movers, count); });
  if (rc) return rc;
  return L("evict_move", [&] {
    // (with nothing to move, what lies past the lengths)
    const dim3 g(moves.x ? moves.x : 64, moves.y);
    hipLaunchKernelGGL(evict_move<true>, g, dim3(256), 0, st, d, page_table, movers, count, out, left, (u32x4*)cache);
  });
}
