// Latent attention over a paged cache for gfx950: the append with its rotation,
// and the absorbed form for single tokens (or a few a sequence).
//
//   q_lat[h] = w_kv[h, :dn]^T q_nope[h]                      (absorb)
//   s_j = scale (q_lat . c_j + rotate(q_pe) . k_j)           (split over the tokens)
//   o_lat = sum_j softmax(s)_j c_j                           (joined in the last kernel)
//   o[h] = w_kv[h, dn:] o_lat[h]                             (up)
//
// All heads of a sequence read the same cache row, once, as key and as value.
// Sequences that share a prefix read it together: its rows are then those of all of them
// (latent_split over the prefix and over each sequence's own tokens, in one launch or two, or
// latent_prefix for both; the parts are joined alike).  Where the tokens' weights are gathered,
// latent_weigh forms them from the scores, once the rows' sums are known.
//
// q_lat is rounded to the operand type, as the MFMA takes it (with weights it enters as two
// such numbers: a score's rounding is one of its weight); the probabilities
// and o_lat, fp32, enter their products as the sum of two bf16 numbers (the cache's
// bytes leave the matrix instructions idle; with probabilities of eight bits o was off
// by 0.0025 of its norm at 64 sequences of up to 8192 tokens, now by 0.0023, of which
// its own rounding is 0.0017 and q_lat's most of the rest).
#include "latent_decode.hpp"

namespace ah {

// ------------------------------------------------------------------- append
struct AppDims {
  int N, H, dn, dr, dc, page, pages, rope, inter;
  int64_t cs, ks, qs[2];
  unsigned blocks_c;  // workgroups of the cache part, the others rotate q
};

// Four pairs of one row: elements 8 u .. 8 u + 7 (interleaved) or 4 u .. + 3 of both halves.
// y1 receives the same, or with LO what y0's rounding left out.
template <typename T> struct Vec4;
template <> struct Vec4<bf16> { typedef bf16x4 t; };
template <> struct Vec4<float> { typedef f32x4 t; };
template <typename T, bool LO = false>
__device__ __forceinline__ void rotate4(const T* x, const float* cr, const float* sr, int u, int dr, bool inter,
                                        T* y0, T* y1) {
  typedef typename Vec4<T>::t v4;
  const int a = inter ? 8 * u : 4 * u, b = inter ? a + 4 : a + dr / 2;
  const v4 lo = *reinterpret_cast<const v4*>(x + a), hi = *reinterpret_cast<const v4*>(x + b);
  const f32x4 c = *reinterpret_cast<const f32x4*>(cr + 4 * u), s = *reinterpret_cast<const f32x4*>(sr + 4 * u);
  f32x4 o0, o1;
  if (inter) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float p = (float)lo[2 * j], q = (float)lo[2 * j + 1], r = (float)hi[2 * j], t = (float)hi[2 * j + 1];
      o0[2 * j] = p * c[j] - q * s[j];
      o0[2 * j + 1] = q * c[j] + p * s[j];
      o1[2 * j] = r * c[2 + j] - t * s[2 + j];
      o1[2 * j + 1] = t * c[2 + j] + r * s[2 + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p = (float)lo[j], q = (float)hi[j];
      o0[j] = p * c[j] - q * s[j];
      o1[j] = q * c[j] + p * s[j];
    }
  }
  if (y0) {
    store4(y0 + a, o0);
    store4(y0 + b, o1);
  }
  if (y1) {
    store4(y1 + a, LO ? rounding<T>(o0) : o0);
    store4(y1 + b, LO ? rounding<T>(o1) : o1);
  }
}

// One 16-byte piece to copy or four pairs to rotate a thread.  Bound by the copy: 8192
// tokens with 16 heads of 128 + 64 and 512 latents, 23 to 24 us for 123 MB, 5.2 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void latent_append(AppDims d, const T* __restrict__ c_kv, const T* __restrict__ k_pe,
                                                     const int64_t* __restrict__ slots,
                                                     const int32_t* __restrict__ pos, const float* __restrict__ cos,
                                                     const float* __restrict__ sin, const T* __restrict__ q,
                                                     T* __restrict__ cache, T* __restrict__ k_out,
                                                     T* __restrict__ q_out) {
  constexpr int V = 16 / (int)sizeof(T);
  if (blockIdx.x < d.blocks_c) {
    const unsigned per = d.dc / V + d.dr / 8, i = blockIdx.x * 256 + threadIdx.x;
    const unsigned t = i / per, u = i % per;
    if (t >= (unsigned)d.N) return;
    const int64_t slot = cache ? slots[t] : -1;
    T* row = slot >= 0 && slot < (int64_t)d.page * d.pages ? cache + slot * (d.dc + d.dr) : nullptr;
    if (u < (unsigned)(d.dc / V)) {
      if (row) *reinterpret_cast<u32x4*>(row + u * V) = *reinterpret_cast<const u32x4*>(c_kv + t * d.cs + u * V);
    } else {
      const int64_t p = min(max(pos[t], 0), d.rope - 1);
      rotate4(k_pe + t * d.ks, cos + p * (d.dr / 2), sin + p * (d.dr / 2), (int)(u - d.dc / V), d.dr, d.inter,
              row ? row + d.dc : nullptr, k_out ? k_out + (int64_t)t * d.dr : nullptr);
    }
  } else {
    const unsigned per = d.dn / V + d.dr / 8, i = (blockIdx.x - d.blocks_c) * 256 + threadIdx.x;
    const unsigned r = i / per, u = i % per, t = r / d.H, h = r % d.H;
    if (t >= (unsigned)d.N) return;
    const T* x = q + t * d.qs[0] + h * d.qs[1];
    T* y = q_out + (int64_t)r * (d.dn + d.dr);
    if (u < (unsigned)(d.dn / V)) {
      *reinterpret_cast<u32x4*>(y + u * V) = *reinterpret_cast<const u32x4*>(x + u * V);
    } else {
      const int64_t p = min(max(pos[t], 0), d.rope - 1);
      rotate4(x + d.dn, cos + p * (d.dr / 2), sin + p * (d.dr / 2), (int)(u - d.dn / V), d.dr, d.inter, y + d.dn,
              (T*)nullptr);
    }
  }
}

// ------------------------------------------------------------------- decode
// q_lat [B n, H, dc | rotated q_pe]: a head, 16 query tokens and 64 latent
// columns a workgroup, 16 columns a wave; one more column block rotates.  Latency: 4 to
// 6 us with 4 to 64 sequences of 16 heads (4 MB of weights).  With LO each row is
// followed by what its rounding left out (bf16; zeros in fp32 have no place).
template <typename T, bool LO>
__global__ __launch_bounds__(256) void latent_absorb(DecDims d, const T* __restrict__ q, const T* __restrict__ w_kv,
                                                     const int32_t* __restrict__ kv_lens,
                                                     const float* __restrict__ cos, const float* __restrict__ sin,
                                                     T* __restrict__ qa) {
  constexpr int V = 16 / (int)sizeof(T), LW = 64 + V, LQ = 128 + V;
  __shared__ __attribute__((aligned(16))) T sw[128 * LW];
  __shared__ __attribute__((aligned(16))) T sq[16 * LQ];
  const int h = blockIdx.x, c0 = 64 * blockIdx.y, r0 = 16 * blockIdx.z, R = d.B * d.n, wide = d.dc + d.dr;
  constexpr int NR = LO ? 2 : 1;
  if (c0 >= d.dc) {
    for (int e = threadIdx.x; e < 16 * (d.dr / 8); e += 256) {
      const int r = r0 + e / (d.dr / 8), u = e % (d.dr / 8);
      if (r >= R) break;
      const T* x = q + r / d.n * d.qs[0] + r % d.n * d.qs[1] + h * d.qs[2] + d.dn;
      T* y = qa + ((int64_t)r * d.H + h) * NR * wide + d.dc;
      if (cos) {
        const int64_t at = (int64_t)pre_len(d, r / d.n) + dec_len(d, kv_lens, r / d.n) - d.n + r % d.n;
        const int64_t p = min(max(at, (int64_t)0), (int64_t)d.rope - 1);
        rotate4<T, LO>(x, cos + p * (d.dr / 2), sin + p * (d.dr / 2), u, d.dr, d.inter, y, LO ? y + wide : (T*)nullptr);
      } else {
        float t[8];
        load8(x + 8 * u, t);
        store8(y + 8 * u, t);
        if constexpr (LO) {
#pragma unroll
          for (int j = 0; j < 8; ++j) t[j] = 0.f;
          store8(y + wide + 8 * u, t);
        }
      }
    }
    return;
  }
  const int KP = (d.dn + 31) / 32 * 32;  // k padded to whole steps with zeros on both sides
  for (int e = threadIdx.x; e < KP * (64 / V); e += 256) {
    const int k = e / (64 / V), c = e % (64 / V) * V;
    u32x4 x = {0, 0, 0, 0};
    if (k < d.dn && c0 + c < d.dc)
      x = *reinterpret_cast<const u32x4*>(w_kv + ((int64_t)h * (d.dn + d.dv) + k) * d.dc + c0 + c);
    *reinterpret_cast<u32x4*>(sw + k * LW + c) = x;
  }
  for (int e = threadIdx.x; e < 16 * (KP / V); e += 256) {
    const int r = min(r0 + e / (KP / V), R - 1), k = e % (KP / V) * V;
    u32x4 x = {0, 0, 0, 0};
    if (k < d.dn) x = *reinterpret_cast<const u32x4*>(q + r / d.n * d.qs[0] + r % d.n * d.qs[1] + h * d.qs[2] + k);
    *reinterpret_cast<u32x4*>(sq + e / (KP / V) * LQ + k) = x;
  }
  __syncthreads();
  const f32x4 z = tile_mma<T, true, false>(zero4(), sw, LW, sq, LQ, 16 * wave_id(), 0, KP);
  const int r = r0 + tile_col(), c = c0 + 16 * wave_id() + tile_row(0);
  if (r < R && c < d.dc) {
    T* y = qa + ((int64_t)r * d.H + h) * NR * wide + c;
    store4(y, z);
    if constexpr (LO) store4(y + wide, rounding<T>(z));
  }
}

template <typename T, int DC, int MT, int NW, bool SCORED, bool FRONT>
__global__ __launch_bounds__(64 * NW) void latent_split(DecDims d, const T* __restrict__ qa,
                                                        const T* __restrict__ cache, const int32_t* __restrict__ table,
                                                        const int32_t* __restrict__ kv_lens,
                                                        const int32_t* __restrict__ own, int own_most,
                                                        float* __restrict__ part, float* __restrict__ stat,
                                                        float* __restrict__ olat, float* __restrict__ score) {
  __shared__ __attribute__((aligned(1024))) SplitLds<T, DC, NW> lds;
  split_tokens<T, DC, MT, NW, SCORED, FRONT>(d, lds, blockIdx.x, blockIdx.y, blockIdx.z, qa, cache, table, kv_lens, own,
                                      own_most, part, stat, olat, score);
}
// Prefixes and own tokens in one launch, where both are small (a launch less): the
// prefixes' workgroups, then the others.  (One grid with the larger of both in each dimension has
// empty workgroups; 6000 of them, each of which waits for a CU's LDS, took 45 us.)
template <typename T, int DC, int MT, int NW, bool SCORED>
__global__ __launch_bounds__(64 * NW) void latent_split_both(DecDims f, DecDims d, int units, const T* __restrict__ qa,
                                                             const T* __restrict__ cache,
                                                             const int32_t* __restrict__ prefix_table,
                                                             const int32_t* __restrict__ prefix_lens,
                                                             const int32_t* __restrict__ table,
                                                             const int32_t* __restrict__ kv_lens,
                                                             float* __restrict__ part, float* __restrict__ stat,
                                                             float* __restrict__ olat, float* __restrict__ score) {
  const int of_front = f.splits * f.groups * units;
  const bool front = (int)blockIdx.x < of_front;
  const int own_most = d.table * d.page, id = blockIdx.x - (front ? 0 : of_front);
  if (front) d = f;
  __shared__ __attribute__((aligned(1024))) SplitLds<T, DC, NW> lds;
  split_tokens<T, DC, MT, NW, SCORED, true>(d, lds, id % d.splits, id / d.splits % d.groups, id / d.splits / d.groups, qa,
                                      cache, front ? prefix_table : table, front ? prefix_lens : kv_lens,
                                      front ? kv_lens : nullptr, own_most, part, stat, olat, front ? nullptr : score);
}
// o_lat [B n H, dc]: the splits of a row joined.  16 `ways` threads take 64
// columns of a row, thread group g the splits g, g + ways, ...; the groups join
// through LDS.  (With few rows and many splits the parts are spread over the card
// this way: 4 sequences of 32768 tokens, 16 heads: 16 MB of parts.)
template <bool FRONT>
__global__ __launch_bounds__(256) void latent_join(DecDims d, int ways, const float* __restrict__ part,
                                                   const float* __restrict__ stat,
                                                   const int32_t* __restrict__ kv_lens, float* __restrict__ olat) {
  __shared__ f32x4 sa[256];
  __shared__ float sm[256], ss[256];
  const int per = 16 * ways, cb = (d.dc + 63) / 64, rows = d.n * d.H, tid = threadIdx.x;
  const int64_t u = (int64_t)blockIdx.x * (256 / per) + tid / per;  // (row, block of columns)
  const int g = tid % per / 16, c = (int)(u % cb) * 64 + 4 * (tid & 15);
  const int64_t row = u / cb;
  const bool ok = row < (int64_t)d.B * rows && c < d.dc;
  float m = -INFINITY, sum = 0.f;
  f32x4 x = zero4();
  if (ok) {
    const int b = (int)(row / rows);
    const Parts<FRONT> ps(d, kv_lens, b);
    const int64_t at = (int64_t)b * d.slots * rows + row % rows, own = at + (int64_t)ps.skip * rows;
    int s = g;
    for (; s < ps.front; s += ways) m = fmaxf(m, stat[2 * (at + (int64_t)s * rows)]);
    for (; s < ps.all; s += ways) m = fmaxf(m, stat[2 * (own + (int64_t)s * rows)]);
    const float ref = m == -INFINITY ? 0.f : m;
    auto take = [&](int64_t a) {
      const float w = fast_exp2(stat[2 * a] - ref);
      sum += w * stat[2 * a + 1];
      x += w * *reinterpret_cast<const f32x4*>(part + a * d.dc + c);
    };
    s = g;
#pragma unroll 4
    for (; s < ps.front; s += ways) take(at + (int64_t)s * rows);
#pragma unroll 4
    for (; s < ps.all; s += ways) take(own + (int64_t)s * rows);
  }
  sa[tid] = x;
  sm[tid] = m;
  ss[tid] = sum;
  __syncthreads();
  if (!ok || g) return;
  for (int i = 1; i < ways; ++i) m = fmaxf(m, sm[tid + 16 * i]);
  const float ref = m == -INFINITY ? 0.f : m;
  x = zero4();
  sum = 0.f;
  for (int i = 0; i < ways; ++i) {
    const float w = fast_exp2(sm[tid + 16 * i] - ref);
    sum += w * ss[tid + 16 * i];
    x += w * sa[tid + 16 * i];
  }
  store4(olat + row * d.dc + c, x * (sum == 0.f ? 0.f : 1.f / sum));
}

// weights[b, j] += sum over the query rows of p_j = 2^(s_j - lse), from the scores that
// latent_split left; the n newest tokens' begin here.  Each token's sum is made by one
// wave in a fixed order: over the row tiles, then across the 16 rows of a tile.  A
// workgroup forms the rows' lse from the parts' statistics, sixteen lanes a row (the rows that
// a tile is padded with, and those that see nothing, get infinity), and goes over
// kWeighTiles tiles.  Reads 4 bytes a row and token, where latent_split read 1152 a token (64
// sequences of 8192 tokens, 16 heads: 25 MB, 7 us beside the up-projection's 8).
constexpr int kWeighTiles = 16, kMostRows = 4096;
// Sum over the sixteen lanes of a row, in each of them, by rotations within it (through LDS, as __shfl_xor goes, a
// tile's 16 of them took as long as its scores).
template <int CTRL> __device__ __forceinline__ float row_turn(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_sum16(float v) {
  return row_turn<0x121>(row_turn<0x122>(row_turn<0x124>(row_turn<0x128>(v))));
}
struct Weigh {
  int row_tiles, first;  // row tiles of a sequence; latent_up's grid x where its workgroups begin
  const float* score;
  const float* shift;  // corrections of the rows' sums over their prefixes (latent_prefix_join), or NULL
  float* weights;
  int64_t stride;
};
template <bool FRONT>
__device__ __forceinline__ void latent_weigh(const DecDims& d, const Weigh& x, const float* __restrict__ stat,
                                             const int32_t* __restrict__ kv_lens, float* lse) {
  const int per = (int)(((int64_t)d.table * d.page + 16 * kWeighTiles - 1) / (16 * kWeighTiles));
  const int64_t id = ((int64_t)(blockIdx.x - x.first) * gridDim.y + blockIdx.y) * gridDim.z + blockIdx.z;
  const int b = (int)(id / per), chunk = (int)(id % per), rows = d.n * d.H, lane = lane_id();
  if (b >= d.B) return;
  const int len = dec_len(d, kv_lens, b);
  if (16 * kWeighTiles * chunk >= len) return;
  const Parts<FRONT> ps(d, kv_lens, b);
  for (int r = threadIdx.x >> 4; r < 16 * x.row_tiles; r += 16) {
    float m = -INFINITY, sum = 0.f;
    if (r < rows) {
      const float* st = stat + 2 * ((int64_t)b * d.slots * rows + r);
      float shift = 0.f;
      if (x.shift) {
#pragma unroll
        for (int k = 0; k < 8; ++k) shift += x.shift[((int64_t)b * rows + r) * 8 + k];
      }
      for (int s = lane & 15; s < ps.all; s += 16) {
        float2 a = *reinterpret_cast<const float2*>(st + 2 * (int64_t)ps.slot(s) * rows);
        if (s < ps.front) a.x += shift;
        const float mn = fmaxf(m, a.x);
        sum = mn > -INFINITY ? sum * fast_exp2(m - mn) + a.y * fast_exp2(a.x - mn) : sum + a.y;
        m = mn;
      }
    }
#pragma unroll
    for (int k = 1; k < 16; k *= 2) {
      const float mo = __shfl_xor(m, k), so = __shfl_xor(sum, k), mn = fmaxf(m, mo);
      sum = mn > -INFINITY ? sum * fast_exp2(m - mn) + so * fast_exp2(mo - mn) : sum + so;
      m = mn;
    }
    // (a NaN among a row's scores stays one, also where a part has no other: its maximum is -inf then, its sum NaN)
    if ((lane & 15) == 0) lse[r] = sum == 0.f ? INFINITY : m + fast_log2(sum);
  }
  __syncthreads();
  const int tiles = (d.table * d.page + 15) / 16;
  f32x4 w[kWeighTiles / 4];
#pragma unroll
  for (int i = 0; i < kWeighTiles / 4; ++i) w[i] = zero4();
  const int t0 = kWeighTiles * chunk + wave_id();
#pragma unroll 2
  for (int g = 0; g < x.row_tiles; ++g) {
    const float z = lse[16 * g + (lane & 15)];
    const float* sc = x.score + ((((int64_t)b * x.row_tiles + g) * tiles) * 64 + lane) * 4;
    f32x4 s[kWeighTiles / 4];
#pragma unroll
    for (int i = 0; i < kWeighTiles / 4; ++i)  // (tiles past the last repeat it)
      s[i] = *reinterpret_cast<const f32x4*>(sc + (int64_t)min(t0 + 4 * i, (len - 1) / 16) * 256);
#pragma unroll
    for (int i = 0; i < kWeighTiles / 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) w[i][r] += fast_exp2(s[i][r] - z);
  }
#pragma unroll
  for (int i = 0; i < kWeighTiles / 4; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) w[i][r] = row_sum16(w[i][r]);
    const int j = 16 * (t0 + 4 * i) + tile_row(lane & 3);
    const float add = (lane & 2) ? ((lane & 1) ? w[i][3] : w[i][2]) : ((lane & 1) ? w[i][1] : w[i][0]);
    float* to = x.weights + b * x.stride + j;
    if ((lane & 15) < 4 && j < len) *to = (j < len - d.n ? *to : 0.f) + add;
  }
}

// o: 16 query tokens of a head times 64 rows of its value projection a
// workgroup, 16 a wave.  With JOIN it joins the splits itself (up to kUpSplits of
// them): where that is a few dozen loads a thread, a launch less is worth more than
// the same parts read once instead of dv / 64 times.  Latency: 5 to 8 us without the join.
// With SCORED the workgroups from grid x `x.first` on gather the tokens' weights instead.
constexpr int kUpSplits = 64;
template <typename T, bool JOIN, bool SCORED, bool FRONT>
__global__ __launch_bounds__(256) void latent_up(DecDims d, const T* __restrict__ w_kv, const float* __restrict__ olat,
                                                 const float* __restrict__ part, const float* __restrict__ stat,
                                                 const int32_t* __restrict__ kv_lens, T* __restrict__ o, Weigh x) {
  constexpr int V = 16 / (int)sizeof(T), LD = 512 + V, PARTS = sizeof(T) == 2 ? 2 : 1, KS = 16;
  __shared__ __attribute__((aligned(16))) T so[PARTS][16 * LD];
  __shared__ float sw[JOIN ? 16 : 1][kUpSplits];
  static_assert(sizeof(so) >= (kMostRows + 64) * sizeof(float), "a float for each row of a sequence's row tiles");
  if (SCORED && (int)blockIdx.x >= x.first) return latent_weigh<FRONT>(d, x, stat, kv_lens, reinterpret_cast<float*>(so));
  const int h = blockIdx.x, v0 = 64 * blockIdx.y, r0 = 16 * blockIdx.z, R = d.B * d.n, KP = (d.dc + 31) / 32 * 32;
  const int vr = v0 + 16 * wave_id(), rows = d.n * d.H;
  const T* w = w_kv + ((int64_t)h * (d.dn + d.dv) + d.dn + min(vr + (lane_id() & 15), d.dv - 1)) * d.dc;
  typename M16<T>::frag wf[KS];  // all of this wave's weights in flight before the rows are waited for
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    const int k = 32 * t + 8 * (lane_id() >> 4);
    wf[t] = ld_frag(k < d.dc ? w + k : (const T*)lat_zeros);
  }
  if constexpr (JOIN) {  // the splits' weights: sixteen threads a row
    const int r = min(r0 + (int)(threadIdx.x >> 4), R - 1), b = r / d.n, g = threadIdx.x & 15;
    const Parts<FRONT> ps(d, kv_lens, b);
    const float* st = stat + 2 * ((int64_t)b * d.slots * rows + r % d.n * d.H + h);
    float m = -INFINITY, sum = 0.f, ms[kUpSplits / 16], ls[kUpSplits / 16];
#pragma unroll
    for (int i = 0; i < kUpSplits / 16; ++i) {
      const int s = g + 16 * i;
      ms[i] = s < ps.all ? st[2 * (int64_t)ps.slot(s) * rows] : -INFINITY;
      ls[i] = s < ps.all ? st[2 * (int64_t)ps.slot(s) * rows + 1] : 0.f;
      m = fmaxf(m, ms[i]);
    }
#pragma unroll
    for (int x = 8; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < kUpSplits / 16; ++i) {
      ms[i] = fast_exp2(ms[i] - ref);
      sum += ms[i] * ls[i];
    }
#pragma unroll
    for (int x = 8; x; x >>= 1) sum += __shfl_xor(sum, x);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < kUpSplits / 16; ++i) sw[threadIdx.x >> 4][g + 16 * i] = ms[i] * inv;
    __syncthreads();
  }
#pragma unroll 4
  for (int e = threadIdx.x; e < 16 * (KP / 4); e += 256) {
    const int r = e / (KP / 4), c = e % (KP / 4) * 4;
    f32x4 x = zero4();
    if (c < d.dc && r0 + r < R) {
      if constexpr (JOIN) {
        const int b = (r0 + r) / d.n;
        const Parts<FRONT> ps(d, kv_lens, b);
        const float* p = part + ((int64_t)b * d.slots * rows + (r0 + r) % d.n * d.H + h) * d.dc + c;
        // (a loop for each kind of parts: with their slots chosen in one the loads were not sent eight at a time)
        int s = 0;
        if constexpr (FRONT) {
#pragma unroll 8
          for (; s < ps.front; ++s) x += sw[r][s] * *reinterpret_cast<const f32x4*>(p + (int64_t)s * rows * d.dc);
          p += (int64_t)ps.skip * rows * d.dc;
        }
#pragma unroll 8
        for (; s < ps.all; ++s) x += sw[r][s] * *reinterpret_cast<const f32x4*>(p + (int64_t)s * rows * d.dc);
      } else {
        x = *reinterpret_cast<const f32x4*>(olat + ((int64_t)(r0 + r) * d.H + h) * d.dc + c);
      }
    }
    store4(&so[0][r * LD + c], x);
    if constexpr (PARTS == 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] -= (float)(T)x[j];
      store4(&so[PARTS - 1][r * LD + c], x);
    }
  }
  __syncthreads();
  if (vr >= d.dv) return;
  f32x4 acc = zero4();
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    if (32 * t < KP) {
#pragma unroll
      for (int p = 0; p < PARTS; ++p)
        acc = M16<T>::mma(wf[t], ld_frag(&so[p][(lane_id() & 15) * LD + 32 * t + 8 * (lane_id() >> 4)]), acc);
    }
  }
  const int r = r0 + tile_col(), v = vr + tile_row(0);
  if (r < R && v < d.dv) store4(o + ((int64_t)r * d.H + h) * d.dv + v, acc);
}

// ------------------------------------------------------------------ host
static int app_check(const atomic_latent_append_args* a) {
  if (!a) return ATOMIC_ERR_NULL;
  if (int rc = latent_widths_check(a->dn, a->dr, a->dtype)) return rc;
  if (a->dc < 8 || a->dc > 512 || a->dc % 8 || a->tokens < 1 || a->heads < 0 || a->page < 1 || a->pages < 1 ||
      a->rope_rows < 1 || (a->interleaved != 0 && a->interleaved != 1))
    return ATOMIC_ERR_SHAPE;
  if (!whole_pieces({a->c_stride, a->k_stride, a->q_stride[0], a->q_stride[1]}, a->dtype)) return ATOMIC_ERR_SHAPE;
  // pieces are counted in 31 bits (a launch of 2^31 pieces moves 64 GB)
  const int v = a->dtype == ATOMIC_BF16 ? 8 : 4;
  if ((int64_t)a->tokens * (a->dc / v + a->dr / 8) > INT32_MAX - 256 ||
      (int64_t)a->tokens * a->heads > INT32_MAX ||
      (int64_t)a->tokens * a->heads * (a->dn / v + a->dr / 8) > INT32_MAX - 256)
    return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}

// `least`: pages that a table has to have
static int dec_check(const atomic_latent_decode_args* a, int least = 1) {
  if (!a) return ATOMIC_ERR_NULL;
  if (int rc = latent_widths_check(a->dn, a->dr, a->dtype)) return rc;
  if (a->dv < 8 || a->dv > 128 || a->dv % 8 || a->dc < 8 || a->dc > 512 || a->dc % 8 || a->batch < 1 ||
      a->tokens < 1 || a->heads < 1 || (int64_t)a->tokens * a->heads > 4096 || a->page < 1 || a->pages < 1 ||
      a->table_pages < least || (a->interleaved != 0 && a->interleaved != 1))
    return ATOMIC_ERR_SHAPE;
  // grid dimensions and token numbers
  if (a->batch > 65535 || (int64_t)a->batch * a->tokens > 65535 * 16 ||
      (int64_t)a->table_pages * a->page > (1 << 30))
    return ATOMIC_ERR_SHAPE;
  if (!whole_pieces({a->q_stride[0], a->q_stride[1], a->q_stride[2]}, a->dtype)) return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}

static int shared_check(const atomic_latent_shared_args* a) {
  if (!a) return ATOMIC_ERR_NULL;
  if (int rc = dec_check(&a->dec, 0)) return rc;
  const atomic_latent_decode_args* c = &a->dec;
  if (a->prefixes < 0 || a->prefix_pages < 0 || (a->scored != 0 && a->scored != 1) ||
      (int64_t)a->prefix_pages * c->page > (1 << 30) ||
      (c->table_pages < 1 && (a->prefixes == 0 || a->prefix_pages < 1)))  // no token at all
    return ATOMIC_ERR_SHAPE;
  // positions behind a prefix are 32-bit
  if ((int64_t)a->prefix_pages * c->page + (int64_t)c->table_pages * c->page > INT32_MAX) return ATOMIC_ERR_SHAPE;
  // the rows that read a prefix are one grid dimension
  if (a->prefixes && (c->batch % a->prefixes ||
                      (int64_t)(c->batch / a->prefixes) * c->tokens * c->heads > (1 << 20)))
    return ATOMIC_ERR_SHAPE;
  if (a->scored && a->weights_stride < (int64_t)c->table_pages * c->page) return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}

// Rows a workgroup of latent_split takes, in tiles of 16.
static int dec_row_tiles(int64_t rows, int dtype) {
  return rows <= 16 ? 1 : rows <= 32 || dtype != ATOMIC_BF16 ? 2 : 4;
}

// (`wide`: four waves a workgroup whatever its row tiles, as in latent_prefix.  `fit`: no second round for a few
// workgroups.)
static DecDims dec_dims(const atomic_latent_decode_args* a, int units, int share, int table, int mt, bool wide = false,
                        bool fit = false) {
  DecDims d{a->batch, a->tokens, a->heads, a->dn, a->dr, a->dv, a->dc, a->page, a->pages, table,
            a->rope_rows, a->interleaved, 0, 0, 0, a->scale, {a->q_stride[0], a->q_stride[1], a->q_stride[2]},
            share, 0, 0, 1, 0, 0, 1, 0, 0, nullptr};
  const int64_t rows = (int64_t)share * d.n * d.H;
  const int rt = 16 * mt, tile = mt == 4 || wide ? 64 : 32;
  d.groups = (int)((rows + rt - 1) / rt);
  // As many workgroups as the card holds at once if every sequence were as long as
  // its table (the host does not know the lengths, so a table wider than the sequences
  // costs parallelism: 64 of 1024 tokens, 16 heads, whole calls: 42 us with a table as
  // wide, 89 with one of 8192 tokens, 293 with one of 131072): two a CU with two waves each in bf16, else one (the tiles' LDS).
  // Split and join together, us: 64 sequences of up to 8192 tokens, 16 heads: 116 in
  // splits of 512, 103 of 1024; 4 of 32768: 42 of 256 or 512, 56 of 128; 8 of 4096
  // with 64 rows: 33 of 128, 36 of 256, 46 of 64; one of 777: 18 of 32, 22 of 128.
  const int64_t slots = mt == 4 || wide || a->dtype != ATOMIC_BF16 ? 256 : 512;
  const int64_t most = (int64_t)d.table * d.page, want = (most * units * d.groups + slots - 1) / slots;
  const int64_t chunk = want < tile ? tile : want > kDecChunk ? kDecChunk : want;
  d.chunk = (int)((chunk + tile - 1) / tile * tile);
  d.splits = (int)((most + d.chunk - 1) / d.chunk);
  // Whole tiles can make a few workgroups more than the card holds, and those a second round: longer splits then.
  // (Us: 625 float32 rows over 3211 tokens, in 260 workgroups 117, in 170 90; five prefixes of 3445 tokens, 525 rows each,
  // in 270 70, in 225 54; 94 sequences of 500 tokens, 36 heads, with weights, in 282 74, in 188 54.)
  const int64_t wg = (int64_t)d.splits * units * d.groups;
  if (fit && wg > slots && 2 * wg < 3 * slots) {
    for (int c = d.chunk + tile; c <= kDecChunk; c += tile) {
      const int64_t s = (most + c - 1) / c;
      if (s * units * d.groups > slots) continue;
      d.chunk = c;
      d.splits = (int)s;
      break;
    }
  }
  d.slots = d.splits;
  return d;
}

// A call's launches over the sequences' own tokens and over the prefixes (with `front.splits` 0 there is none).
struct DecPlan {
  DecDims own, front;
  int own_tiles, front_tiles;  // row tiles of a workgroup
  bool many;                   // the prefixes' rows are many: latent_prefix takes them
  bool both;                   // one launch for both
};
static DecPlan dec_plan(const atomic_latent_decode_args* a, int prefixes, int prefix_pages, bool scored) {
  DecPlan p{};
  p.own_tiles = dec_row_tiles((int64_t)a->tokens * a->heads, a->dtype);
  // (without prefixes and weights as it always was: a sum's bits follow its splits)
  p.own = dec_dims(a, a->batch, 1, a->table_pages, p.own_tiles, false, prefixes || scored);
  const int qn = scored && a->dtype == ATOMIC_BF16 ? 2 : 1;
  p.own.qn = qn;
  if (!prefixes) return p;
  const int share = a->batch / prefixes;
  p.front_tiles = dec_row_tiles((int64_t)share * a->tokens * a->heads, a->dtype);
  // (float32, whose matrix instructions are the bound: four waves, with one tile in LDS, where there are tokens
  // enough to use them.  Us: 624 rows over 2952 tokens 63, with two tiles and waves 151; 931 rows over 2 tokens and
  // the own tokens of 49 sequences 50, with two, then in one launch, 34.)
  if (a->dtype != ATOMIC_BF16 && p.front_tiles == 2 && (int64_t)share * a->tokens * a->heads > 32 &&
      (int64_t)prefix_pages * a->page >= 512)
    p.front_tiles = 4;
  p.front = dec_dims(a, prefixes, share, prefix_pages, p.front_tiles, false, true);
  DecDims many = p.front;
  const DecDims own = dec_dims(a, a->batch, 1, a->table_pages, p.own_tiles, true);
  if (a->dtype == ATOMIC_BF16 && prefix_plan(many, prefixes, own)) {
    const int64_t wgs = (int64_t)own.splits * own.groups * a->batch;  // one grid dimension for both
    p.many = wgs <= (1 << 30);
    if (p.many) {
      p.front = many;
      p.own = own;
    }
  }
  // One launch for both costs less than what the own tokens lose by the prefix's row tiles while they are few: in bf16
  // up to some 262144 of them (32 rows over 4000 tokens, 32 sequences of own tokens, us, in one launch and in two: 22.9
  // and 29 of 1024, 42 and 47 of 4096, 69 and 73 of 8192, 126 and 126 of 16384), in float32, bound by the products that an empty row tile has too,
  // up to some 4096 (32 rows over 777, 16 of 4096: 192 and 76; 24 rows over 1501, 6 of 130: 21 and 34).
  p.both = !p.many && p.front_tiles <= 2 && p.front.splits && p.own.splits &&
           (int64_t)p.front.splits * p.front.groups * prefixes <= (1 << 29) &&
           (int64_t)a->batch * a->table_pages * a->page <=
               (a->dtype != ATOMIC_BF16 && p.own_tiles != p.front_tiles ? 4096 : 262144);
  if (p.both && p.own_tiles != p.front_tiles) {
    p.own_tiles = p.front_tiles;
    p.own = dec_dims(a, a->batch, 1, a->table_pages, p.own_tiles, false, true);
  }
  p.own.qn = p.front.qn = p.many ? 2 : qn;
  p.own.slot0 = p.front.splits;
  if (p.many) p.own.part0 = p.front.splits;
  p.own.slots = p.front.slots = p.own.splits + p.front.splits;
  p.own.pre_share = p.front.share;
  p.own.pre_chunk = p.front.chunk;
  p.own.pre_splits = p.front.splits;
  p.own.pre_most = prefix_pages * a->page;
  return p;
}

// Whether latent_up joins the splits: at most 48 loads a thread, in steps of eight
// (25 loads: 14.6 us against 7.4 + 7.2 of two launches, 64: 25.7 against 9 + 10).
static bool dec_up_joins(const DecDims& d) {
  const int64_t rows = (int64_t)d.B * d.n < 16 ? (int64_t)d.B * d.n : 16;
  return d.slots > 1 && d.slots <= kUpSplits && d.slots * ((rows * d.dc / 4 + 255) / 256) <= 48;
}
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }
// What a call leaves in its workspace, part after part.
struct DecSpace {
  size_t qa, olat, stat, part, front, shift, score, all;
};
static DecSpace dec_space(const DecPlan& p, int prefixes, int dtype, bool scored) {
  const DecDims& d = p.own;
  const size_t rows = (size_t)d.B * d.n * d.H, es = dtype == ATOMIC_BF16 ? 2 : 4;
  const size_t parts = d.slots > 1 ? rows * (d.slots - d.part0) : 0;  // one split needs no parts
  const size_t tiles = (size_t)d.groups * p.own_tiles * (((size_t)d.table * d.page + 15) / 16);
  DecSpace s;
  s.qa = 0;
  s.olat = s.qa + up256(rows * (d.dc + d.dr) * es * d.qn);
  s.stat = s.olat + up256(rows * d.dc * sizeof(float));
  s.part = s.stat + up256((scored || d.slots > 1 ? rows * d.slots : 0) * 2 * sizeof(float));
  s.front = s.part + up256(parts * d.dc * sizeof(float));
  s.shift = s.front + (p.many ? up256(prefix_bytes(p.front, prefixes)) : 0);
  s.score = s.shift + (p.many && scored ? up256(rows * 8 * sizeof(float)) : 0);
  s.all = s.score + (scored ? (size_t)d.B * tiles * 256 * sizeof(float) : 0);
  return s;
}

}  // namespace ah

using namespace ah;

extern "C" int atomic_latent_append(const atomic_latent_append_args* a, const void* c_kv, const void* k_pe,
                                    const int64_t* slots, const int32_t* positions, const float* cos,
                                    const float* sin, const void* q, void* cache, void* k_out, void* q_out,
                                    void* stream) {
  if (int rc = app_check(a)) return rc;
  if (!k_pe || !positions || !cos || !sin || (cache && (!c_kv || !slots)) || (q && (!q_out || a->heads < 1)))
    return ATOMIC_ERR_NULL;
  if (!aligned16({c_kv, k_pe, cos, sin, q, cache, k_out, q_out})) return ATOMIC_ERR_SHAPE;
  AppDims d{a->tokens, q ? a->heads : 1, a->dn, a->dr, a->dc, a->page, a->pages, a->rope_rows, a->interleaved,
            a->c_stride, a->k_stride, {a->q_stride[0], a->q_stride[1]}, 0};
  const int v = a->dtype == ATOMIC_BF16 ? 8 : 4;
  d.blocks_c = (unsigned)(((int64_t)d.N * (d.dc / v + d.dr / 8) + 255) / 256);
  const unsigned bq = q ? (unsigned)(((int64_t)d.N * d.H * (d.dn / v + d.dr / 8) + 255) / 256) : 0;
  const hipStream_t st = (hipStream_t)stream;
  Launch L{a->profile, st};
  return L("latent_append", [&] {
    if (a->dtype == ATOMIC_BF16)
      hipLaunchKernelGGL((latent_append<bf16>), dim3(d.blocks_c + bq), dim3(256), 0, st, d, (const bf16*)c_kv,
                         (const bf16*)k_pe, slots, positions, cos, sin, (const bf16*)q, (bf16*)cache, (bf16*)k_out,
                         (bf16*)q_out);
    else
      hipLaunchKernelGGL((latent_append<float>), dim3(d.blocks_c + bq), dim3(256), 0, st, d, (const float*)c_kv,
                         (const float*)k_pe, slots, positions, cos, sin, (const float*)q, (float*)cache,
                         (float*)k_out, (float*)q_out);
  });
}

struct DecPtrs {
  const void *q, *w_kv, *cache;
  const int32_t *prefix_table, *prefix_lens, *table, *lens;
  const float *cos, *sin;
  float* weights;
  int64_t weights_stride;
  void *o, *ws;
};

// Where a call's parts lie in its workspace.
template <typename T> struct DecParts {
  T* qa;
  float *olat, *stat, *part, *score;
};

// latent_split over the prefixes (`front`) or the own tokens, or both where the plan says so.
template <typename T, int DC, bool SCORED>
static void launch_split(const DecPlan& plan, int prefixes, bool front, hipStream_t st, const DecPtrs& p,
                         const DecParts<T>& x) {
  const DecDims &d = plan.own, &f = plan.front;
  const int own_most = d.table * d.page;
  auto go = [&](auto m) {
    constexpr int MT = decltype(m)::value, NW = MT == 4 ? 4 : 2;
    if constexpr (MT <= 2) {
      if (plan.both) {
        const dim3 grid((unsigned)(d.splits * d.groups * d.B + f.splits * f.groups * prefixes));
        hipLaunchKernelGGL((latent_split_both<T, DC, MT, NW, SCORED>), grid, dim3(64 * NW), 0, st, f, d, prefixes, x.qa,
                           (const T*)p.cache, p.prefix_table, p.prefix_lens, p.table, p.lens, x.part, x.stat, x.olat,
                           x.score);
        return;
      }
    }
    if (front)
      hipLaunchKernelGGL((latent_split<T, DC, MT, NW, SCORED, true>),
                         dim3((unsigned)f.splits, (unsigned)f.groups, (unsigned)prefixes), dim3(64 * NW), 0, st, f, x.qa,
                         (const T*)p.cache, p.prefix_table, p.prefix_lens, p.lens, own_most, x.part, x.stat, x.olat,
                         (float*)nullptr);
    else
      hipLaunchKernelGGL((latent_split<T, DC, MT, NW, SCORED, false>),
                         dim3((unsigned)d.splits, (unsigned)d.groups, (unsigned)d.B), dim3(64 * NW), 0, st, d, x.qa,
                         (const T*)p.cache, p.table, p.lens, (const int32_t*)nullptr, 0, x.part, x.stat, x.olat, x.score);
  };
  const int mt = front ? plan.front_tiles : plan.own_tiles;
  if (mt == 1) go(IntC<1>());
  else if (mt == 2) go(IntC<2>());
  else go(IntC<4>());
}

template <typename T, bool SCORED>
static int dec_run(const atomic_latent_decode_args* a, int prefixes, int prefix_pages, const DecPtrs& p,
                   hipStream_t st) {
  DecPlan plan = dec_plan(a, prefixes, prefix_pages, SCORED);
  plan.own.pre_lens = p.prefix_lens;
  const DecDims& d = plan.own;
  const DecSpace at = dec_space(plan, prefixes, a->dtype, SCORED);
  Launch L{a->profile, st};
  char* ws = (char*)p.ws;
  const DecParts<T> x{(T*)(ws + at.qa), (float*)(ws + at.olat), (float*)(ws + at.stat), (float*)(ws + at.part),
                      SCORED ? (float*)(ws + at.score) : nullptr};
  const unsigned rt = (unsigned)((d.B * d.n + 15) / 16);
  int rc = L("latent_absorb", [&] {
    const dim3 grid((unsigned)d.H, (unsigned)((d.dc + 63) / 64 + 1), rt);
    if constexpr (sizeof(T) == 2) {
      if (d.qn == 2) {
        hipLaunchKernelGGL((latent_absorb<T, true>), grid, dim3(256), 0, st, d, (const T*)p.q, (const T*)p.w_kv, p.lens,
                           p.cos, p.sin, x.qa);
        return;
      }
    }
    hipLaunchKernelGGL((latent_absorb<T, false>), grid, dim3(256), 0, st, d, (const T*)p.q, (const T*)p.w_kv, p.lens,
                       p.cos, p.sin, x.qa);
  });
  if (rc) return rc;
  auto split = [&](bool front) {
    if (d.dc <= 256) launch_split<T, 256, SCORED>(plan, prefixes, front, st, p, x);
    else launch_split<T, 512, SCORED>(plan, prefixes, front, st, p, x);
  };
  if (plan.both) {
    rc = L("latent_split_both", [&] { split(true); });
    if (rc) return rc;
  }
  PrefixCall pre{plan.front, d, prefixes, plan.own_tiles, (const bf16*)x.qa, (const bf16*)p.cache, p.prefix_table,
                 p.prefix_lens, p.table, p.lens, x.part, x.stat, x.olat, x.score, ws + at.front};
  if (plan.many) {
    rc = L("latent_prefix", [&] { launch_prefix(pre, SCORED, st); });
    if (rc) return rc;
  }
  if (plan.front.splits && !plan.both && !plan.many) {
    rc = L("latent_split (prefix)", [&] { split(true); });
    if (rc) return rc;
  }
  if (d.splits && !plan.both && !plan.many) {
    rc = L("latent_split", [&] { split(false); });
    if (rc) return rc;
  }
  const bool joins = !plan.many && dec_up_joins(d);
  float* shift = plan.many && SCORED ? (float*)(ws + at.shift) : nullptr;
  if (plan.many) {
    rc = L("latent_prefix_join", [&] { launch_prefix_join(pre, st, shift); });
    if (rc) return rc;
  } else if (d.slots > 1 && !joins) {
    int ways = 1;  // about four splits a thread
    while (ways < 16 && 4 * ways < d.slots) ways *= 2;
    const int64_t units = (int64_t)d.B * d.n * d.H * ((d.dc + 63) / 64);
    rc = L("latent_join", [&] {
      auto go = [&](auto f) {
        hipLaunchKernelGGL(latent_join<decltype(f)::value != 0>, dim3((unsigned)((units * ways + 15) / 16)), dim3(256), 0,
                           st, d, ways, x.part, x.stat, p.lens, x.olat);
      };
      if (prefixes) go(IntC<1>());
      else go(IntC<0>());
    });
    if (rc) return rc;
  }
  const Weigh wx{d.groups * plan.own_tiles, d.H, x.score, shift, p.weights, p.weights_stride};
  unsigned more = 0;  // the weights' workgroups
  const unsigned gy = (unsigned)((d.dv + 63) / 64);
  if (SCORED && d.splits) {
    const int64_t per = ((int64_t)d.table * d.page + 16 * kWeighTiles - 1) / (16 * kWeighTiles);
    more = (unsigned)((per * d.B + gy * rt - 1) / (gy * rt));
  }
  return L("latent_up", [&] {
    auto go = [&](auto j, auto f) {
      hipLaunchKernelGGL((latent_up<T, decltype(j)::value != 0, SCORED, decltype(f)::value != 0>),
                         dim3((unsigned)d.H + more, gy, rt), dim3(256), 0, st, d, (const T*)p.w_kv, x.olat, x.part,
                         x.stat, p.lens, (T*)p.o, wx);
    };
    if (!joins && (!SCORED || !prefixes)) go(IntC<0>(), IntC<0>());
    else if (!joins) go(IntC<0>(), IntC<SCORED>());
    else if (prefixes) go(IntC<1>(), IntC<1>());
    else go(IntC<1>(), IntC<0>());
  });
}

extern "C" size_t atomic_latent_decode_workspace_size(const atomic_latent_decode_args* a) {
  if (dec_check(a) != ATOMIC_OK) return 0;
  return dec_space(dec_plan(a, 0, 0, false), 0, a->dtype, false).all;
}

extern "C" int atomic_latent_decode(const atomic_latent_decode_args* a, const void* q, const void* w_kv,
                                    const void* cache, const int32_t* page_table, const int32_t* kv_lens,
                                    const float* cos, const float* sin, void* o, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (int rc = dec_check(a)) return rc;
  if (!q || !w_kv || !cache || !page_table || !kv_lens || !o || !cos != !sin) return ATOMIC_ERR_NULL;
  if (cos && a->rope_rows < 1) return ATOMIC_ERR_SHAPE;
  if (!aligned16({q, w_kv, cache, cos, sin, o})) return ATOMIC_ERR_SHAPE;
  if (!workspace || workspace_bytes < atomic_latent_decode_workspace_size(a) || !aligned16({workspace}))
    return ATOMIC_ERR_WORKSPACE;
  ws_tag_clobber(workspace, atomic_latent_decode_workspace_size(a));
  const DecPtrs p{q, w_kv, cache, nullptr, nullptr, page_table, kv_lens, cos, sin, nullptr, 0, o, workspace};
  return a->dtype == ATOMIC_BF16 ? dec_run<bf16, false>(a, 0, 0, p, (hipStream_t)stream)
                                 : dec_run<float, false>(a, 0, 0, p, (hipStream_t)stream);
}

extern "C" size_t atomic_latent_decode_shared_workspace_size(const atomic_latent_shared_args* a) {
  if (shared_check(a) != ATOMIC_OK) return 0;
  return dec_space(dec_plan(&a->dec, a->prefixes, a->prefix_pages, a->scored != 0), a->prefixes, a->dec.dtype, a->scored != 0)
      .all;
}

extern "C" int atomic_latent_decode_shared(const atomic_latent_shared_args* a, const void* q, const void* w_kv,
                                           const void* cache, const int32_t* prefix_table, const int32_t* prefix_lens,
                                           const int32_t* page_table, const int32_t* kv_lens, const float* cos,
                                           const float* sin, float* weights, void* o, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  if (int rc = shared_check(a)) return rc;
  if (!q || !w_kv || !cache || !kv_lens || !o || !cos != !sin || (a->dec.table_pages && !page_table) ||
      (a->prefixes && (!prefix_lens || (a->prefix_pages && !prefix_table))) || 
      (a->scored && a->dec.table_pages && !weights))
    return ATOMIC_ERR_NULL;
  if (cos && a->dec.rope_rows < 1) return ATOMIC_ERR_SHAPE;
  if (!aligned16({q, w_kv, cache, cos, sin, o})) return ATOMIC_ERR_SHAPE;
  const size_t bytes = atomic_latent_decode_shared_workspace_size(a);
  if (!workspace || workspace_bytes < bytes || !aligned16({workspace})) return ATOMIC_ERR_WORKSPACE;
  ws_tag_clobber(workspace, bytes);
  const DecPtrs p{q,   w_kv, cache, prefix_table, prefix_lens,       page_table, kv_lens,
                  cos, sin,  weights, a->weights_stride, o, workspace};
  const auto run = [&](auto t) {
    typedef decltype(t) T;
    return a->scored ? dec_run<T, true>(&a->dec, a->prefixes, a->prefix_pages, p, (hipStream_t)stream)
                     : dec_run<T, false>(&a->dec, a->prefixes, a->prefix_pages, p, (hipStream_t)stream);
  };
  return a->dec.dtype == ATOMIC_BF16 ? run(bf16()) : run(float());
}
