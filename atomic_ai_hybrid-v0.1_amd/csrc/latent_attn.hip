// Latent attention in its expanded form for gfx950: forward and backward over
// k_nope and v as the up-projection leaves them ([.., H, dn + dv]) and the
// rotated key that all heads share.
//
//   s_ij = scale (q_nope_i . k_nope_j + q_pe_i . k_pe_j)     visible j only
//   o_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i)
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = do_i . o_i
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dk_pe_j summed over the heads
//
// Scores and probabilities live in registers only (latent.hpp); the score gradients
// too, unless the backward's first large kernel leaves them for its second (bf16, up
// to 4 GB).  p and ds are rounded to the operand type for the second product, as its
// MFMA takes them; everything else (scores, the running maximum and sum, lse, delta,
// every accumulator) is fp32.  In bf16 that rounding is as large as the result's own:
// of the norm, o is off by 0.0021 to 0.0023 and a gradient by 0.0023 to 0.0024 (0.0027
// where a query sees five keys or fewer) where their own roundings are 0.0017.  p and ds
// as two bf16 numbers each would leave only the results' roundings and make 8 MFMAs more
// of a 32 x 32 tile's 20 in the forward, 20 more of 40 in latent_bwd_dkv, and the score
// gradients in memory twice as large.
//
// A query that sees one key (always the first) has p = 1 whatever its score, so ds = 0.
// Formed as do . v - do . o it would be what the two sums' roundings leave (the one in
// the order of the matrix instructions, the other in latent_delta's), 1e-7 of the terms
// where the gradient is zero: its ds is therefore formed with a weight of zero.
//
// Masked places are replaced, not weighted, so a masked score may be anything; a
// masked value enters a product with a weight of zero, as in any tiled or plain form,
// so an infinity or NaN in a later token of a causal sequence can reach the queries
// before it.  Rows past the lengths are never read.
#include <cfloat>

#include "latent.hpp"

namespace ah {

constexpr int kAhead = 2;  // groups of fragments that the backward reads ahead
struct LatDims {
  int B, T, S, H, dn, dr, dv, causal, blocks;  // blocks: row (or token) blocks of a head
  float scale;
  int64_t qs[3], ks[3], ps[2], gs[3];  // strides of q, kv, k_pe, do
};

// Workgroup -> (head of the batch, block of its rows).  The heads are dealt over the
// XCDs, so that a head's other operand is in one L2 (workgroups go round the eight in
// turn), and within an XCD the first blocks of all heads come first: with causal they
// are the longest, and the shortest fill the gaps at the end.  (Head by head, three
// rounds of 32 workgroups end with the third's longest: 340 us instead of 296 for the
// forward of 48 heads of 4096.)
__device__ __forceinline__ void lat_map(const LatDims& d, int& b, int& h, int& blk) {
  const int heads = d.B * d.H, per = heads % 8 == 0 ? heads / 8 : heads;
  const int x = heads % 8 == 0 ? blockIdx.x / 8 : blockIdx.x;
  const int bh = (heads % 8 == 0 ? blockIdx.x % 8 * per : 0) + x % per;
  blk = x / per;
  b = bh / d.H;
  h = bh % d.H;
}
__device__ __forceinline__ int clamp_len(const int32_t* p, int b, int most) {
  return p ? min(max(p[b], 0), most) : most;
}

// A row of two spans (w0 elements from src0, then from element W0 on w1 from src1)
// as register fragments, padded with zeros: this lane's row at src0 / src1.
template <typename T, int W0, int W1>
__device__ __forceinline__ void row_frags(typename M32<T>::frag (&f)[(W0 + W1) / 16], const T* src0, int w0,
                                          const T* src1, int w1) {
  const int h8 = 8 * (lane_id() >> 5);
#pragma unroll
  for (int s = 0; s < (W0 + W1) / 16; ++s) {
    const int k = 16 * s + h8;
    f[s] = zero_frag<T>();
    if (16 * s < W0) {
      if (k < w0) f[s] = ld_frag(src0 + k);
    } else if (k - W0 < w1) {
      f[s] = ld_frag(src1 + k - W0);
    }
  }
}

// Keep a value in the accumulator half of the register file (a kernel of one wave a
// SIMD has 256 registers in each).
template <typename F> __device__ __forceinline__ void in_accum(F& x) { asm volatile("" : "+a"(x)); }

// What rounding to T leaves out.
template <typename T> __device__ __forceinline__ f32x4 rounding(f32x4 x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] -= (float)(T)x[j];
  return x;
}

// Token of register r of a score tile (from its first token).
__device__ __forceinline__ int reg_row(int r) { return 8 * (r >> 2) + 4 * (lane_id() >> 5) + (r & 3); }

// ------------------------------------------------------------------ forward
// 128 query rows of a head a workgroup, 32 a wave, against tiles of 64 tokens (32 in
// fp32) that go straight to LDS, one tile ahead; one barrier a tile.  Two workgroups a
// CU, so two waves a SIMD with 256 registers each: one's MFMAs run beside the other's
// softmax.  (Eight waves on one tile, the two of a SIMD half a tile apart, took half the
// tiles out of L2 and still lost, by the longer workgroups' tails: 9 % at B8 T4096 H6,
// 7 % at B2 T8192 H16, 1 % at B1 T8192 H16, both timed in turn when that was changed.)
//
// Bound by the matrix instructions and the clock that the card holds under them: at
// B2 T8192 H16, 128/64/128, causal the matrix pipes are busy for 59 % of the kernel's
// cycles at 1.4 to 1.7 GHz, 655 to 690 us, 1.0 to 1.05 PF/s, where the library's product
// of two 8192 x 8192 matrices reaches 1.21.
//
// With `parts` > 1 the keys of a row block are divided over that many workgroups
// (few row blocks against many keys); each leaves its accumulators, reference and
// sum, which latent_fwd_join joins.
template <typename T, int DN, int DR, int DV>
__global__ __launch_bounds__(256, 2) void latent_fwd(LatDims d, int parts, const T* __restrict__ q, const T* __restrict__ kv,
                                                    const T* __restrict__ kpe, const int32_t* __restrict__ q_lens,
                                                    const int32_t* __restrict__ kv_lens, T* __restrict__ o,
                                                    float* __restrict__ lse, T* __restrict__ rest,
                                                    float* __restrict__ pacc, float* __restrict__ pstat) {
  constexpr int KN = DN / 16, KS = (DN + DR) / 16, NT = DV / 32, TK = sizeof(T) == 2 ? 64 : 32, NS = TK / 32;
  constexpr int FG = sizeof(T) == 2 ? 2 : 1, FL = 2;  // fragments are read four MFMAs ahead (fp32: sixteen)
  typedef LTile<T, DN> LN;
  typedef LTile<T, DR> LR;
  typedef LTile<T, DV> LV;
  typedef typename M32<T>::frag frag;
  constexpr int OR = TK * LN::ROWB, OV = OR + TK * LR::ROWB, STAGE = OV + TK * LV::ROWB;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  int b, h, blk;
  lat_map(d, b, h, blk);
  const int part = blk % parts;
  blk = (d.blocks - 1 - blk) / parts;  // with causal the long rows first (`parts` divides `blocks`)
  const int ql = clamp_len(q_lens, b, d.T), kl = clamp_len(kv_lens, b, d.S), off = kl - ql;
  const int w0 = 128 * blk + 32 * wave_id();  // this wave's first row
  const int row = w0 + (lane_id() & 31);
  const int last = min(128 * blk + 127, ql - 1);  // the workgroup's last row
  int begin = 0, end = kl;                          // keys that any row sees
  if (d.causal) end = min(end, last + off + 1);
  if (last < 128 * blk) end = 0;
  if (parts > 1) {
    const int tiles = (max(end, 0) + TK - 1) / TK;
    begin = (int)((int64_t)tiles * part / parts) * TK;
    end = min(end, (int)((int64_t)tiles * (part + 1) / parts) * TK);
  }
  const T* qr = q + b * d.qs[0] + (int64_t)max(min(row, ql - 1), 0) * d.qs[1] + h * d.qs[2];
  const T* kb = kv + b * d.ks[0] + h * d.ks[2];
  StageDma<RowDma<T, DN, TK, 4>, RowDma<T, DR, TK, 4>, RowDma<T, DV, TK, 4>> dma;
  dma.a.init(kb, d.ks[1], d.dn);
  dma.b.init(kpe + b * d.ps[0], d.ps[1], d.dr);
  dma.c.init(kb + d.dn, d.ks[1], d.dv);
  dma.ob = OR;
  dma.oc = OV;
  frag qf[KS];
  row_frags<T, DN, DR>(qf, qr, d.dn, qr + d.dn, d.dr);
  // (a scale of zero as the smallest number: a masked score stays infinite; a negative one changes q's sign)
  const float c2 = d.scale == 0.f ? FLT_MIN : fabsf(d.scale) * kLog2e;
  if (d.scale < 0.f) {
#pragma unroll
    for (int t = 0; t < KS; ++t) qf[t] = -qf[t];
  }
  f32x16 acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = zero16();
  float m = -INFINITY, sum = 0.f;  // reference (of c2 times the scores, see kLag) and this lane's part of the sum
  const uint32_t l0 = lds_addr(lds);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the query: no later wait for it drains the tiles
  const uint32_t bn = LN::row_base(), br = LR::row_base(), bv = LV::col_base();
  f32x16 s[NS];
  // Scores of a tile, masked, and a new reference where one is far above its row's.
  // `to`: where the tile that `dma` aims at goes, sent for along the way (past the last
  // key, zeros).
  auto scores = [&](uint32_t at, int k0, uint32_t to) {
    uint32_t an = at + bn, ar = at + OR + br;
    asm volatile("" : "+v"(an), "+v"(ar));
#pragma unroll
    for (int i = 0; i < NS; ++i) s[i] = zero16();
    in_groups<KS * NS, FG, FL, 0, frag>(
        [&](int j) {
          const int t = j / NS, i = j % NS;
          return t < KN ? LN::row(an, 32 * i, 16 * t) : LR::row(ar, 32 * i, 16 * (t - KN));
        },
        [&](int j, frag a) { s[j % NS] = M32<T>::mma(a, qf[j / NS], s[j % NS]); },
        [&](int j) { dma.at_slot(j, KS * NS, to); });
    if (k0 + TK > kl || (d.causal && k0 + TK - 1 > w0 + off)) {
      const int seen = min(kl, d.causal ? row + off + 1 : kl) - k0 - reg_row(0);
#pragma unroll
      for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          int lim = seen;  // (each compare by itself: chained, their conditions fill the scalar registers)
          asm volatile("" : "+v"(lim));
          s[i][r] = 32 * i + 8 * (r >> 2) + (r & 3) < lim ? s[i][r] : -INFINITY;
        }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[i][r]);
    top *= c2;
    if (__any(top > m + kLag)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top), fade = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
      m = mn;
      sum *= fade;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[n][r] *= fade;
    }
  };
  // The tile's probabilities and their products with the values; the second half's
  // exponentials run beside the first half's products.
  auto values = [&](uint32_t at) {
    uint32_t av = at + OV + bv;
    asm volatile("" : "+v"(av));
    const float ref = m == -INFINITY ? 0.f : -m;  // a row that has seen nothing yet: every p is exp2(-inf) = 0
    frag p[2 * NS];
    auto quad = [&](int i, int k) {  // four tokens
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = fast_exp2(__builtin_fmaf(s[i][4 * k + j], c2, ref));
        sum += x;
        p[2 * i + k / 2][4 * (k & 1) + j] = (T)x;
      }
    };
#pragma unroll
    for (int k = 0; k < 4; ++k) quad(0, k);
    __builtin_amdgcn_sched_barrier(0);
    in_groups<2 * NS * NT, FG, FL, NS == 2 ? 14 : 0, frag>(
        [&](int j) { return LV::col(av, 16 * (j / NT), 32 * (j % NT)); },
        [&](int j, frag a) { acc[j % NT] = M32<T>::mma(a, p[j / NT], acc[j % NT]); },
        [&](int j) {
          if (NS == 2 && j < 4) quad(1, j);
        });
    static_assert(NS == 1 || 2 * NT >= 4, "the second half's probabilities are there in time");
  };
  dma.start(begin, min(kl, end) - 1);
  dma.aim();
  dma.all(l0);
  int k0 = begin, buf = 0;
  auto stage = [&] {
    vm_wait<0>();
    bare_barrier();  // the tile is there, and nobody reads the other one any more
    dma.aim();
  };
  // tiles that this wave's rows see anything of, then those that only the others do
  const int any = w0 >= ql ? 0 : min(end, d.causal ? w0 + 32 + off : kl);
  for (; k0 < any; k0 += TK, buf ^= 1) {
    stage();
    scores(l0 + buf * STAGE, k0, l0 + (buf ^ 1) * STAGE);
    values(l0 + buf * STAGE);
  }
  for (; k0 < end; k0 += TK, buf ^= 1) {
    stage();
    dma.all(l0 + (buf ^ 1) * STAGE);
  }
  vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
  if (row >= d.T) return;
  sum += __shfl_xor(sum, 32);
  const int64_t at = ((int64_t)b * d.H + h) * d.T + row;
  if (parts > 1) {
    const int64_t pr = (int64_t)part * d.B * d.H * d.T + at;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int c = 32 * n + reg_row(r);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = row < ql ? acc[n][r + j] : 0.f;  // (a weight of zero would keep a NaN)
        if (c < d.dv) store4(pacc + pr * d.dv + c, v);
      }
    if (lane_id() < 32) {
      pstat[2 * pr] = row < ql ? m : -INFINITY;
      pstat[2 * pr + 1] = row < ql ? sum : 0.f;
    }
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* orow = o + (((int64_t)b * d.T + row) * d.H + h) * d.dv;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * n + reg_row(r);
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = row < ql ? acc[n][r + j] * inv : 0.f;
      if (c < d.dv) {
        store4(orow + c, v);
        if (rest) store4(rest + (orow - o) + c, rounding<T>(v));
      }
    }
  if (lane_id() < 32) lse[at] = row < ql && sum != 0.f ? m * kLn2 + fast_log2(sum) * kLn2 : -INFINITY;
}

// o and lse of rows whose keys were divided: four columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void latent_fwd_join(LatDims d, int parts, const float* __restrict__ pacc,
                                                       const float* __restrict__ pstat, T* __restrict__ o,
                                                       float* __restrict__ lse, T* __restrict__ rest) {
  const int per = d.dv / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, at = i / per, rows = (int64_t)d.B * d.H * d.T;
  if (at >= rows) return;
  const int c = (int)(i % per) * 4;
  float m = -INFINITY, sum = 0.f;
  for (int p = 0; p < parts; ++p) m = fmaxf(m, pstat[2 * (p * rows + at)]);
  const float ref = m == -INFINITY ? 0.f : m;
  f32x4 x = zero4();
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const float w = fast_exp2(pstat[2 * (p * rows + at)] - ref);
    sum += w * pstat[2 * (p * rows + at) + 1];
    x += w * *reinterpret_cast<const f32x4*>(pacc + (p * rows + at) * d.dv + c);
  }
  const int t = (int)(at % d.T), h = (int)(at / d.T % d.H), b = (int)(at / d.T / d.H);
  const int64_t to = (((int64_t)b * d.T + t) * d.H + h) * d.dv + c;
  x *= sum == 0.f ? 0.f : 1.f / sum;
  store4(o + to, x);
  if (rest) store4(rest + to, rounding<T>(x));
  if (c == 0) lse[at] = sum == 0.f ? -INFINITY : m * kLn2 + fast_log2(sum) * kLn2;
}

// ----------------------------------------------------------------- backward
// Rows of delta and lse a head: whole tiles, so that the rows past the last query
// can hold an lse of infinity (every p of theirs is zero).
__host__ __device__ inline int64_t stat_rows(int T) { return (int64_t)(T + 63) / 64 * 64; }

// stat: delta (from o and, in bf16, what its rounding left out: 13 us of B2 T8192 H16's
// 2.8 ms, for a row that sees few keys most of its scores' gradients) and lse in powers
// of two, each [B, H, stat_rows]: sixteen lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void latent_delta(LatDims d, const T* __restrict__ o, const T* __restrict__ rest,
                                                    const T* __restrict__ dout,
                                                    const float* __restrict__ lse, const int32_t* __restrict__ q_lens,
                                                    float* __restrict__ stat) {
  const int64_t TP = stat_rows(d.T), j = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);  // (b, t, h)
  if (j >= d.B * TP * d.H) return;
  const int h = (int)(j % d.H), t = (int)(j / d.H % TP), b = (int)(j / d.H / TP);
  const int64_t at = ((int64_t)b * d.H + h) * TP + t, half = d.B * TP * d.H;
  if (t >= clamp_len(q_lens, b, d.T)) {
    if ((threadIdx.x & 15) == 0) {
      stat[at] = 0.f;
      stat[half + at] = INFINITY;
    }
    return;
  }
  const int64_t i = ((int64_t)b * d.T + t) * d.H + h;
  const T* g = dout + b * d.gs[0] + t * d.gs[1] + h * d.gs[2];
  float s = 0.f;
  for (int c = 8 * (threadIdx.x & 15); c < d.dv; c += 128) {
    float x[8], y[8];
    load8(o + i * d.dv + c, x);
    if (rest) {
      load8(rest + i * d.dv + c, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] += y[j];
    }
    load8(g + c, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) s += x[j] * y[j];
  }
#pragma unroll
  for (int x = 8; x; x >>= 1) s += __shfl_xor(s, x);
  if ((threadIdx.x & 15) == 0) {
    // (a query that sees nothing has lse = -infinity; all of its places are masked)
    stat[at] = s;
    stat[half + at] = lse[((int64_t)b * d.H + h) * d.T + t] * kLog2e;
  }
}

// dq where the score gradients are not kept (fp32, and bf16 above kMostDs): 128 query
// rows of a head a workgroup, 32 a wave, against tiles of tokens staged as in the
// forward; scores and their gradients once more.  B2 T8192 H16 bf16: 1068 us, where
// latent_bwd_dq_ds takes 531 and its score gradients cost latent_bwd_dkv 195.
template <typename T, int DN, int DR, int DV>
__global__ __launch_bounds__(256, 1) void latent_bwd_dq(
    LatDims d, const T* __restrict__ q, const T* __restrict__ kv, const T* __restrict__ kpe,
    const int32_t* __restrict__ q_lens, const int32_t* __restrict__ kv_lens, const float* __restrict__ stat,
    const T* __restrict__ dout, T* __restrict__ dq, int parts, float* __restrict__ pq) {
  constexpr int KN = DN / 16, KS = (DN + DR) / 16, VS = DV / 16, NN = DN / 32, NT = (DN + DR) / 32;
  constexpr int TK = sizeof(T) == 2 ? 64 : 32, NS = TK / 32;
  typedef LTile<T, DN> LN;
  typedef LTile<T, DR> LR;
  typedef LTile<T, DV> LV;
  typedef typename M32<T>::frag frag;
  constexpr int OR = TK * LN::ROWB, OV = OR + TK * LR::ROWB, STAGE = OV + TK * LV::ROWB;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  int b, h, blk;
  lat_map(d, b, h, blk);
  const int part = blk % parts;
  blk = (d.blocks - 1 - blk) / parts;
  const int ql = clamp_len(q_lens, b, d.T), kl = clamp_len(kv_lens, b, d.S), off = kl - ql;
  const int w0 = 128 * blk + 32 * wave_id();
  const int row = w0 + (lane_id() & 31);
  const int last = min(128 * blk + 127, ql - 1);
  int begin = 0, end = kl;
  if (d.causal) end = min(end, last + off + 1);
  if (last < 128 * blk) end = 0;
  if (parts > 1) {
    const int tiles = (max(end, 0) + TK - 1) / TK;
    begin = (int)((int64_t)tiles * part / parts) * TK;
    end = min(end, (int)((int64_t)tiles * (part + 1) / parts) * TK);
  }
  const int rowc = max(min(row, ql - 1), 0);
  const T* qr = q + b * d.qs[0] + (int64_t)rowc * d.qs[1] + h * d.qs[2];
  const T* kb = kv + b * d.ks[0] + h * d.ks[2];
  StageDma<RowDma<T, DN, TK, 4>, RowDma<T, DR, TK, 4>, RowDma<T, DV, TK, 4>> dma;
  dma.a.init(kb, d.ks[1], d.dn);
  dma.b.init(kpe + b * d.ps[0], d.ps[1], d.dr);
  dma.c.init(kb + d.dn, d.ks[1], d.dv);
  dma.ob = OR;
  dma.oc = OV;
  frag qf[KS], gf[VS];
  row_frags<T, DN, DR>(qf, qr, d.dn, qr + d.dn, d.dr);
  row_frags<T, DV, 0>(gf, dout + b * d.gs[0] + (int64_t)rowc * d.gs[1] + h * d.gs[2], d.dv, (const T*)nullptr, 0);
  const int64_t at = ((int64_t)b * d.H + h) * stat_rows(d.T) + rowc;
  // (a row of one key: an lse of infinity makes its p zero)
  const bool one = (d.causal ? min(kl, row + off + 1) : kl) == 1;
  const float dl = stat[at], l2 = one ? INFINITY : stat[(int64_t)d.B * d.H * stat_rows(d.T) + at];
  f32x16 acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = zero16();
  const float c2 = d.scale * kLog2e;
  const uint32_t l0 = lds_addr(lds);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  const int past = begin < end ? end - 1 : -1;  // the last key wanted
  dma.aim_at(begin, past);
  dma.all(l0);
  int k0 = begin, buf = 0;
  uint32_t to;         // where the next tile goes
  auto stage = [&] {  // this tile is there; the next one (past the last, zeros) is sent for along the way
    vm_wait<0>();
    bare_barrier();
    to = l0 + (buf ^ 1) * STAGE;
    dma.aim_at(k0 + TK, past);
  };
  // one tile, its halves a phase apart as in latent_bwd_dkv
  auto step = [&](auto masked) {
    const uint32_t at = l0 + buf * STAGE;
    uint32_t rn = at + LN::row_base(), rr = at + OR + LR::row_base(), rv = at + OV + LV::row_base();
    uint32_t cn = at + LN::col_base(), cr = at + OR + LR::col_base();
    asm volatile("" : "+v"(rn), "+v"(rr), "+v"(rv), "+v"(cn), "+v"(cr));
    const int seen = min(kl, d.causal ? row + off + 1 : kl) - k0;
    f32x16 s[NS], g[NS];
    frag ds[NS][2];
    if constexpr (sizeof(T) == 2) {  // (left alone, half of them change files and back in every tile: 1201 -> 1093 us at B2 T8192 H16)
#pragma unroll
      for (int n = 0; n < NT; ++n) in_accum(acc[n]);
    }
    constexpr int M1 = KS + VS, M2 = 2 * NT;
    auto row_at = [&](int i, int j) {
      return j < KN ? LN::row(rn, 32 * i, 16 * j)
                    : j < KS ? LR::row(rr, 32 * i, 16 * (j - KN)) : LV::row(rv, 32 * i, 16 * (j - KS));
    };
    auto score = [&](int i, int j, frag a) {
      if (j == 0) s[i] = zero16();
      if (j == KS) g[i] = zero16();
      if (j < KS) s[i] = M32<T>::mma(a, qf[j], s[i]);
      else g[i] = M32<T>::mma(a, gf[j - KS], g[i]);
    };
    auto col_at = [&](int i, int j) {
      const int t = j / NT, n = j % NT, r = 32 * i + 16 * t;
      return n < NN ? LN::col(cn, r, 32 * n) : LR::col(cr, r, 32 * (n - NN));
    };
    auto grad = [&](int i, int j, frag a) { acc[j % NT] = M32<T>::mma(a, ds[i][j / NT], acc[j % NT]); };
    auto prob = [&](int i, int k) {  // four tokens
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * k + j;
        float y = fast_exp2(s[i][r] * c2 - l2) * (g[i][r] - dl);
        if constexpr (decltype(masked)::value) y = 32 * i + reg_row(r) < seen ? y : 0.f;
        ds[i][k / 2][4 * (k & 1) + j] = (T)y;
      }
    };
    if constexpr (NS == 2) {
      constexpr int G = M1 % 4 || M2 % 4 ? (M1 % 5 || M2 % 5 ? 2 : 5) : 4;
      static_assert(M1 % G == 0 && M2 % G == 0, "whole groups");
      in_groups<2 * M1 + 2 * M2, G, kAhead, 6, frag>(
          [&](int j) {
            return j < 2 * M1 ? row_at(j / M1, j % M1) : col_at((j - 2 * M1) / M2, (j - 2 * M1) % M2);
          },
          [&](int j, frag a) {
            if (j < 2 * M1) score(j / M1, j % M1, a);
            else grad((j - 2 * M1) / M2, (j - 2 * M1) % M2, a);
          },
          [&](int j) {
            dma.at_slot(j, 2 * M1 + 2 * M2, to);
            if (j >= M1 && j < 2 * M1 && (j - M1) % (M1 / 4) == 1 && (j - M1) / (M1 / 4) < 4) prob(0, (j - M1) / (M1 / 4));
            if (M2 >= 8 && j >= 2 * M1 && j < 2 * M1 + M2 && (j - 2 * M1) % (M2 / 4) == 1 && (j - 2 * M1) / (M2 / 4) < 4)
              prob(1, (j - 2 * M1) / (M2 / 4));
            if (M2 < 8 && j >= 2 * M1 && j < 2 * M1 + 4) prob(1, j - 2 * M1);
          });
    } else {
      dma.all(to);
      in_groups<M1, 4, frag>([&](int j) { return row_at(0, j); }, [&](int j, frag a) { score(0, j, a); });
#pragma unroll
      for (int k = 0; k < 4; ++k) prob(0, k);
      in_groups<M2, 4, frag>([&](int j) { return col_at(0, j); }, [&](int j, frag a) { grad(0, j, a); });
    }
  };
  // tiles that every row of this wave sees whole, those on the diagonal or the last key, those that none sees
  const int whole = w0 >= ql ? 0 : min(end, d.causal ? min(kl, w0 + off + 1) : kl) - TK + 1;
  const int any = w0 >= ql ? 0 : min(end, d.causal ? w0 + 32 + off : kl);
  for (; k0 < whole; k0 += TK, buf ^= 1) {
    stage();
    step(IntC<0>());
  }
  for (; k0 < any; k0 += TK, buf ^= 1) {
    stage();
    step(IntC<1>());
  }
  for (; k0 < end; k0 += TK, buf ^= 1) {
    stage();
    dma.all(to);
  }
  vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
  if (row >= d.T) return;
  T* out = dq + (((int64_t)b * d.T + row) * d.H + h) * (d.dn + d.dr);
  float* po = pq + ((((int64_t)part * d.B + b) * d.T + row) * d.H + h) * (d.dn + d.dr);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * n + reg_row(r);
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = row < ql ? acc[n][r + j] * d.scale : 0.f;
      const int at = 32 * n < DN ? c : d.dn + c - DN;
      if (32 * n < DN ? c < d.dn : c - DN < d.dr) {
        if (parts > 1) store4(po + at, v);
        else store4(out + at, v);
      }
    }
}

// dk, dv: 128 tokens of a head a workgroup, 32 a wave (their keys, values and
// gradient accumulators in registers: one wave a SIMD), against tiles of query
// rows staged as the forward's tokens are, with delta and lse beside them.  The
// rotated key's gradient leaves as this head's part, fp32 [B, H, S, dr].
//
// Four of the backward's five products (scores, dp, dv, dk) run here, bound by the
// matrix instructions and what stands between them (one wave a SIMD): B2 T8192 H16
// causal 1610 to 1670 us, 0.82 to 0.85 PF/s, the matrix pipes busy for 45 % of the cycles.
//
// With DS the score gradients go to memory too, for latent_bwd_dq_ds: [B, H, tiles of
// 64 rows, S, 64] bf16, a token's rows in the order of this kernel's registers
// (ds_piece), 16 bytes a lane as they are, so that a wave writes 4 KB in a row.  (In
// rows of T the 32 tokens of a wave lay a power of two apart: 1710 us instead of
// 1484 at B2 T8192 H16, when that was changed.)  They are the last memory operations of a tile, so the wait for
// the next tile's loads leaves them in flight.
template <typename T, int DN, int DR, int DV, bool DS>
__global__ __launch_bounds__(256, 1) void latent_bwd_dkv(LatDims d, const T* __restrict__ q, const T* __restrict__ kv,
                                                         const T* __restrict__ kpe, const int32_t* __restrict__ q_lens,
                                                         const int32_t* __restrict__ kv_lens,
                                                         const float* __restrict__ stat, const T* __restrict__ dout,
                                                         T* __restrict__ dkv, float* __restrict__ dkp, int parts,
                                                         float* __restrict__ pkv, T* __restrict__ dst) {
  constexpr int KN = DN / 16, KS = (DN + DR) / 16, VS = DV / 16, NN = DN / 32, NK = (DN + DR) / 32, NV = DV / 32;
  constexpr int TQ = sizeof(T) == 2 ? 64 : 32, NS = TQ / 32;
  typedef LTile<T, DN> LN;
  typedef LTile<T, DR> LR;
  typedef LTile<T, DV> LG;
  typedef typename M32<T>::frag frag;
  constexpr int OR = TQ * LN::ROWB, OG = OR + TQ * LR::ROWB, OS = OG + TQ * LG::ROWB, STAGE = OS + 512;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  int b, h, blk;
  lat_map(d, b, h, blk);
  const int part = blk % parts;
  blk /= parts;
  const int ql = clamp_len(q_lens, b, d.T), kl = clamp_len(kv_lens, b, d.S), off = kl - ql;
  const int w0 = 128 * blk + 32 * wave_id();  // this wave's first token
  const int tok = w0 + (lane_id() & 31);
  const int tokc = max(min(tok, kl - 1), 0);
  int first = 0;  // the first query that sees any of the workgroup's tokens
  if (d.causal) first = max(0, 128 * blk - off);
  if (128 * blk >= kl) first = ql;
  first &= ~(TQ - 1);
  int stop = ql;
  if (parts > 1) {
    const int tiles = max(0, (ql - first + TQ - 1) / TQ), from = first;
    first = from + (int)((int64_t)tiles * part / parts) * TQ;
    stop = min(ql, from + (int)((int64_t)tiles * (part + 1) / parts) * TQ);
  }
  const T* qb = q + b * d.qs[0] + h * d.qs[2];
  const T* gb = dout + b * d.gs[0] + h * d.gs[2];
  const T* kr = kv + b * d.ks[0] + (int64_t)tokc * d.ks[1] + h * d.ks[2];
  StageDma<RowDma<T, DN, TQ, 4>, RowDma<T, DR, TQ, 4>, RowDma<T, DV, TQ, 4>> dma;
  dma.a.init(qb, d.qs[1], d.dn);
  dma.b.init(qb + d.dn, d.qs[1], d.dr);
  dma.c.init(gb, d.gs[1], d.dv);
  dma.ob = OR;
  dma.oc = OG;
  // wave 0 brings delta, wave 1 lse (64 rows; an fp32 tile uses half of them)
  const float* sb = stat + ((wave_id() & 1 ? (int64_t)d.B * d.H : 0) + (int64_t)b * d.H + h) * stat_rows(d.T);
  const uint32_t l0 = lds_addr(lds);
  auto aim = [&](int r0, uint32_t to) {
    dma.aim_at(r0, ql - 1);
    if (r0 < ql && wave_id() < 2) dma4_raw(sb + (r0 & ~63) + lane_id(), to + OS + 256 * wave_id());
  };
  frag kf[KS], vf[VS];
  row_frags<T, DN, DR>(kf, kr, d.dn, kpe + b * d.ps[0] + (int64_t)tokc * d.ps[1], d.dr);
  row_frags<T, DV, 0>(vf, kr + d.dn, d.dv, (const T*)nullptr, 0);
  f32x16 ak[NK], av[NV];
#pragma unroll
  for (int n = 0; n < NK; ++n) ak[n] = zero16();
#pragma unroll
  for (int n = 0; n < NV; ++n) av[n] = zero16();
  const float c2 = d.scale * kLog2e;
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  aim(first, l0);
  dma.all(l0);
  int q0 = first, buf = 0;
  uint32_t to;            // where the next tile goes
  bool stored = false;    // the tile before ended with its 2 NS stores
  T* dsp = nullptr;       // this lane's piece of the score gradients at q0 = 0
  if constexpr (DS)
    dsp = dst + (((int64_t)b * d.H + h) * (stat_rows(d.T) / 64) * d.S + min(tok, d.S - 1)) * 64 + 8 * (lane_id() >> 5);
  auto stage = [&] {  // this tile is there; the next one (past the last, zeros) is sent for along the way
    if (DS && stored) vm_wait<2 * NS>();
    else vm_wait<0>();
    bare_barrier();
    to = l0 + (buf ^ 1) * STAGE;
    aim(q0 + TQ, to);
  };
  // One tile.  Its two halves follow each other by a phase: the scores of the
  // second half run beside the first half's exponentials, the gradients of the
  // first beside the second's.  Only the diagonal needs a mask (and a sequence of one
  // key its ds of zero): rows past the last query have an lse of infinity, tokens past
  // the last key are not stored.
  auto step = [&](auto masked) {
    const uint32_t at = l0 + buf * STAGE;
    uint32_t rn = at + LN::row_base(), rr = at + OR + LR::row_base(), rg = at + OG + LG::row_base();
    uint32_t cn = at + LN::col_base(), cr = at + OR + LR::col_base(), cg = at + OG + LG::col_base();
    asm volatile("" : "+v"(rn), "+v"(rr), "+v"(rg), "+v"(cn), "+v"(cr), "+v"(cg));
    const float *sd = (const float*)(lds + buf * STAGE + OS) + (q0 & 63), *sl = sd + 64;
    f32x16 s[NS], g[NS];
    frag p[NS][2], ds[NS][2];
    constexpr int M1 = KS + VS, M2 = 2 * (NV + NK);
    auto row_at = [&](int i, int j) {
      return j < KN ? LN::row(rn, 32 * i, 16 * j)
                    : j < KS ? LR::row(rr, 32 * i, 16 * (j - KN)) : LG::row(rg, 32 * i, 16 * (j - KS));
    };
    auto score = [&](int i, int j, frag a) {
      if (j == 0) s[i] = zero16();
      if (j == KS) g[i] = zero16();
      if (j < KS) s[i] = M32<T>::mma(a, kf[j], s[i]);
      else g[i] = M32<T>::mma(a, vf[j - KS], g[i]);
    };
    auto col_at = [&](int i, int j) {
      const int t = j / (NV + NK), n = j % (NV + NK), r = 32 * i + 16 * t;
      return n < NV ? LG::col(cg, r, 32 * n)
                    : n < NV + NN ? LN::col(cn, r, 32 * (n - NV)) : LR::col(cr, r, 32 * (n - NV - NN));
    };
    auto grad = [&](int i, int j, frag a) {
      const int t = j / (NV + NK), n = j % (NV + NK);
      if (n < NV) av[n] = M32<T>::mma(a, p[i][t], av[n]);
      else ak[n - NV] = M32<T>::mma(a, ds[i][t], ak[n - NV]);
    };
    auto prob = [&](int i, int k) {  // four rows
      const f32x4 l4 = *reinterpret_cast<const f32x4*>(sl + 32 * i + reg_row(4 * k));
      const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + 32 * i + reg_row(4 * k));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * k + j;
        float x = fast_exp2(s[i][r] * c2 - l4[j]), y = x * (g[i][r] - d4[j]);
        if constexpr (decltype(masked)::value) {
          const int end = d.causal ? q0 + 32 * i + reg_row(r) + off : kl - 1;  // the last token that the row sees
          y = end == 0 ? 0.f * (g[i][r] - d4[j]) : y;                          // (a NaN stays one)
          x = tok <= end ? x : 0.f;
          y = tok <= end ? y : 0.f;
        }
        p[i][k / 2][4 * (k & 1) + j] = (T)x;
        ds[i][k / 2][4 * (k & 1) + j] = (T)y;
      }
    };
    auto put = [&](int i) {
      if (tok < d.S) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          *reinterpret_cast<frag*>(dsp + (int64_t)q0 * d.S + 32 * i + 16 * t) = ds[i][t];
      }
    };
    if constexpr (NS == 2) {
      constexpr int G = M1 % 4 || M2 % 4 ? 5 : 4;  // whole groups a phase: a phase's work starts after the one before
      static_assert(M1 % G == 0 && M2 % G == 0, "whole groups");
      in_groups<2 * M1 + 2 * M2, G, kAhead, 6, frag>(
          [&](int j) {
            return j < 2 * M1 ? row_at(j / M1, j % M1) : col_at((j - 2 * M1) / M2, (j - 2 * M1) % M2);
          },
          [&](int j, frag a) {
            if (j < 2 * M1) score(j / M1, j % M1, a);
            else grad((j - 2 * M1) / M2, (j - 2 * M1) % M2, a);
          },
          [&](int j) {
            dma.at_slot(j, DS ? 2 * M1 : 2 * M1 + 2 * M2, to);
            if (j >= M1 && j < 2 * M1 && (j - M1) % (M1 / 4) == 1 && (j - M1) / (M1 / 4) < 4) prob(0, (j - M1) / (M1 / 4));
            if (j >= 2 * M1 && j < 2 * M1 + M2 && (j - 2 * M1) % (M2 / 4) == 1 && (j - 2 * M1) / (M2 / 4) < 4)
              prob(1, (j - 2 * M1) / (M2 / 4));
            if (DS && j >= 2 * M1 && (j - 2 * M1) % M2 == 0) put((j - 2 * M1) / M2);
          });
    } else {
      dma.all(to);
      in_groups<M1, 4, frag>([&](int j) { return row_at(0, j); }, [&](int j, frag a) { score(0, j, a); });
#pragma unroll
      for (int k = 0; k < 4; ++k) prob(0, k);
      in_groups<M2, 4, frag>([&](int j) { return col_at(0, j); }, [&](int j, frag a) { grad(0, j, a); });
    }
  };
  // tiles that this wave's tokens are not visible to, those on the diagonal, the rest
  // (a wave without tokens only keeps the others company)
  for (; q0 < stop && (w0 >= kl || (d.causal && w0 > q0 + TQ - 1 + off)); q0 += TQ, buf ^= 1) {
    stage();
    dma.all(to);
  }
  for (; q0 < stop && (kl == 1 || (d.causal && w0 + 31 > q0 + off)); q0 += TQ, buf ^= 1) {
    stage();
    step(IntC<1>());
    stored = true;
  }
  for (; q0 < stop; q0 += TQ, buf ^= 1) {
    stage();
    step(IntC<0>());
    stored = true;
  }
  vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
  if (tok >= d.S) return;
  const int64_t wide = d.dn + d.dv, at = (((int64_t)b * d.S + tok) * d.H + h) * wide;
  T* out = dkv + at;
  float* po = pkv + (int64_t)part * d.B * d.S * d.H * wide + at;
  float* op = dkp + ((((int64_t)part * d.B + b) * d.H + h) * d.S + tok) * d.dr;
#pragma unroll
  for (int n = 0; n < NK + NV; ++n)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * (n < NK ? n : n - NK) + reg_row(r);
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = tok >= kl ? 0.f : n < NK ? ak[n < NK ? n : 0][r + j] * d.scale : av[n < NK ? 0 : n - NK][r + j];
      if (n >= NN && n < NK) {
        if (c - DN < d.dr) store4(op + c - DN, v);
      } else if (c < (n < NK ? d.dn : d.dv)) {
        const int x = n < NK ? c : d.dn + c;
        if (parts > 1) store4(po + x, v);
        else store4(out + x, v);
      }
    }
}

// Where rows c .. c + 3 (c a multiple of 4) lie in a token's row of the score
// gradients: the piece and the byte in it.  Sixteen rows are two pieces, one of each
// half of the wave: its registers' rows 4 h .. + 3 and 8 + 4 h .. + 3.
__device__ __forceinline__ int ds_piece(int c) { return 2 * (c >> 4) + ((c >> 2) & 1); }
__device__ __forceinline__ int ds_byte(int c) { return 8 * ((c >> 3) & 1); }

// dq from the score gradients that latent_bwd_dkv left: 256 query rows of a head a
// workgroup, 64 a wave, against tiles of 32 tokens, three of them on their way.
// dq^T += k^T ds^T; a fragment of k serves two MFMAs.  Bound by reading the score
// gradients (2 bytes a pair): B2 T8192 H16 causal 540 to 550 us for 2.1 GB, 3.9 TB/s where
// a copy reaches 5.0.
template <int DN, int DR>
__global__ __launch_bounds__(256, 1) void latent_bwd_dq_ds(LatDims d, const bf16* __restrict__ kv,
                                                           const bf16* __restrict__ kpe,
                                                           const int32_t* __restrict__ q_lens,
                                                           const int32_t* __restrict__ kv_lens,
                                                           const bf16* __restrict__ ds, bf16* __restrict__ dq,
                                                           int parts, float* __restrict__ pq) {
  constexpr int NN = DN / 32, NT = (DN + DR) / 32, TK = 32, NB = 4, RG = 2, RW = 32 * RG, RB = 4 * RW;
  typedef LTile<bf16, DN> LN;
  typedef LTile<bf16, DR> LR;
  typedef LTile<bf16, RW> LS;
  typedef bf16x8 frag;
  constexpr int OR = TK * LN::ROWB, OS = OR + TK * LR::ROWB, STAGE = OS + 4 * TK * LS::ROWB;
  __shared__ __attribute__((aligned(1024))) char lds[NB * STAGE];
  int b, h, blk;
  lat_map(d, b, h, blk);
  const int part = blk % parts;
  blk = (d.blocks - 1 - blk) / parts;
  const int ql = clamp_len(q_lens, b, d.T), kl = clamp_len(kv_lens, b, d.S), off = kl - ql;
  const int w0 = RB * blk + RW * wave_id();
  const int last = min(RB * blk + RB - 1, ql - 1);
  int begin = 0, end = kl;
  // (the score gradients are there for whole tiles of 64 rows)
  if (d.causal) end = min(end, (last | 63) + off + 1);
  if (last < RB * blk) end = 0;
  if (parts > 1) {
    const int tiles = (max(end, 0) + TK - 1) / TK;
    begin = (int)((int64_t)tiles * part / parts) * TK;
    end = min(end, (int)((int64_t)tiles * (part + 1) / parts) * TK);
  }
  const bf16* kb = kv + b * d.ks[0] + h * d.ks[2];
  StageDma<RowDma<bf16, DN, TK, 4>, RowDma<bf16, DR, TK, 4>, RowDma<bf16, RW, TK, 1>> dma;
  dma.a.init(kb, d.ks[1], d.dn);
  dma.b.init(kpe + b * d.ps[0], d.ps[1], d.dr);
  // (every wave brings its own rows' score gradients)
  dma.c.init(ds + (((int64_t)b * d.H + h) * (stat_rows(d.T) / 64) + min(w0, ql - 1) / 64) * d.S * 64, 64, RW);
  dma.ob = OR;
  dma.oc = OS + wave_id() * TK * LS::ROWB;
  f32x16 acc[RG][NT];
#pragma unroll
  for (int g = 0; g < RG; ++g)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[g][n] = zero16();
  const uint32_t l0 = lds_addr(lds);
  constexpr int PER = decltype(dma)::N;
  dma.start(begin, end - 1);
#pragma unroll
  for (int i = 0; i < NB - 1; ++i) {
    dma.aim();
    dma.all(l0 + i * STAGE);
  }
  // keys that this wave's rows have gradients for (in whole groups of 32)
  const int any = w0 >= ql ? 0 : min(end, d.causal ? w0 + RW + off : kl);
  const int l = lane_id(), t4 = l & 15, rr = 4 * (l >> 5) + (t4 >> 2);
  int buf = 0;
  for (int k0 = begin; k0 < end; k0 += TK, buf = (buf + 1) % NB) {
    vm_wait<(NB - 2) * PER>();
    bare_barrier();  // the tile is there, and nobody reads the one before it any more
    const uint32_t to = l0 + (buf + NB - 1) % NB * STAGE;
    dma.aim();
    const char* sk = lds + buf * STAGE;
    uint32_t cn = l0 + buf * STAGE + LN::col_base(), cr = l0 + buf * STAGE + OR + LR::col_base();
    asm volatile("" : "+v"(cn), "+v"(cr));
    auto ds_at = [&](int g, int r0) {  // the rows of group g, 16 tokens from r0
      const int c = 32 * g + 16 * ((l >> 4) & 1) + 4 * (t4 & 3);
      typedef __attribute__((address_space(3))) bf16x4* lds_p;
      const char* s = sk + OS + wave_id() * TK * LS::ROWB + ds_byte(c);
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_p)(s + LS::off(r0 + rr, ds_piece(c))));
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_p)(s + LS::off(r0 + 8 + rr, ds_piece(c))));
      return (frag)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
#pragma unroll
    for (int g = 0; g < RG; ++g)
#pragma unroll
      for (int n = 0; n < NT; ++n) in_accum(acc[g][n]);
    if (k0 < any) {
      frag f[2][RG];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int g = 0; g < RG; ++g) f[t][g] = ds_at(g, 16 * t);
      in_groups<2 * NT, 1, 4, 0, frag>(
          [&](int j) {
            const int r = 16 * (j / NT), n = j % NT;
            return n < NN ? LN::col(cn, r, 32 * n) : LR::col(cr, r, 32 * (n - NN));
          },
          [&](int j, frag a) {
#pragma unroll
            for (int g = 0; g < RG; ++g) acc[g][j % NT] = M32<bf16>::mma(a, f[j / NT][g], acc[g][j % NT]);
          },
          [&](int j) { dma.at_slot(j, 2 * NT, to); });
    } else {
      dma.all(to);
    }
  }
  vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const int row = w0 + 32 * g + (l & 31);
    if (row >= d.T) continue;
    const int64_t wide = d.dn + d.dr, at = (((int64_t)b * d.T + row) * d.H + h) * wide;
    bf16* out = dq + at;
    float* po = pq + (int64_t)part * d.B * d.T * d.H * wide + at;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int c = 32 * n + reg_row(r);
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = row < ql ? acc[g][n][r + j] * d.scale : 0.f;
        const int x = n < NN ? c : d.dn + c - DN;
        if (n < NN ? c < d.dn : c - DN < d.dr) {
          if (parts > 1) store4(po + x, v);
          else store4(out + x, v);
        }
      }
  }
}

// What is left to sum, in one launch, four elements a thread and each sum in a fixed
// order: the parts of dk / dv (n1 elements) and of dq (n2; 0 where there is one part),
// and dk_pe from the shares of the heads and of the parts of the queries.
struct FinishJobs {
  int64_t n1, n2;
  unsigned b1, b2;  // workgroups of the first two
  int kparts, qparts;
};
template <typename T>
__global__ __launch_bounds__(256) void latent_bwd_finish(LatDims d, FinishJobs f, const float* __restrict__ pkv,
                                                         const float* __restrict__ pq, const float* __restrict__ dkp,
                                                         T* __restrict__ dkv, T* __restrict__ dq,
                                                         T* __restrict__ dkpe) {
  auto join = [&](unsigned blk, int64_t n, int parts, const float* p, T* out) {
    const int64_t i = ((int64_t)blk * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    f32x4 s = zero4();
#pragma unroll 4
    for (int k = 0; k < parts; ++k) s += *reinterpret_cast<const f32x4*>(p + k * n + i);
    store4(out + i, s);
  };
  if (blockIdx.x < f.b1) return join(blockIdx.x, f.n1, f.kparts, pkv, dkv);
  if (blockIdx.x < f.b1 + f.b2) return join(blockIdx.x - f.b1, f.n2, f.qparts, pq, dq);
  const int64_t i = ((int64_t)(blockIdx.x - f.b1 - f.b2) * 256 + threadIdx.x) * 4, per = (int64_t)d.S * d.dr;
  if (i >= d.B * per) return;
  f32x4 s = zero4();
  for (int k = 0; k < f.kparts; ++k) {
    const float* p = dkp + ((int64_t)k * d.B + i / per) * d.H * per + i % per;
#pragma unroll 4
    for (int h = 0; h < d.H; ++h) s += *reinterpret_cast<const f32x4*>(p + h * per);
  }
  store4(dkpe + i, s);
}

// ------------------------------------------------------------------ host
static int lat_check(const atomic_latent_args* a) {
  if (!a) return ATOMIC_ERR_NULL;
  if (int rc = latent_widths_check(a->dn, a->dr, a->dtype)) return rc;
  if (a->dv < 8 || a->dv > 128 || a->dv % 8 || a->batch < 1 || a->tq < 1 || a->tk < 1 || a->heads < 1 ||
      (a->causal != 0 && a->causal != 1))
    return ATOMIC_ERR_SHAPE;
  // row numbers and lengths stay in 31 bits with room for a block; grids in 31 bits
  if (a->tq > (1 << 30) || a->tk > (1 << 30)) return ATOMIC_ERR_SHAPE;
  const int64_t most = (int64_t)(a->tq > a->tk ? a->tq : a->tk), bh = (int64_t)a->batch * a->heads;
  if (bh > INT32_MAX || bh * ((most + 127) / 128) > INT32_MAX || bh * (stat_rows((int)most) / 16) > INT32_MAX ||
      (int64_t)a->batch * ((a->tk + 15) / 16) * a->dr > INT32_MAX)
    return ATOMIC_ERR_SHAPE;
  const int64_t es = a->dtype == ATOMIC_BF16 ? 2 : 4;
  for (int64_t s : {a->q_stride[1], a->kv_stride[1], a->kpe_stride[1], a->do_stride[1]})
    if (s > kMostRowBytes / es) return ATOMIC_ERR_SHAPE;
  if (!whole_pieces({a->q_stride[0], a->q_stride[1], a->q_stride[2], a->kv_stride[0], a->kv_stride[1],
                     a->kv_stride[2], a->kpe_stride[0], a->kpe_stride[1], a->do_stride[0], a->do_stride[1],
                     a->do_stride[2]}, a->dtype))
    return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}

static LatDims lat_dims(const atomic_latent_args* a) {
  LatDims d{a->batch, a->tq, a->tk, a->heads, a->dn, a->dr, a->dv, a->causal, 0, a->scale, {}, {}, {}, {}};
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a->q_stride[i];
    d.ks[i] = a->kv_stride[i];
    d.gs[i] = a->do_stride[i];
  }
  d.ps[0] = a->kpe_stride[0];
  d.ps[1] = a->kpe_stride[1];
  return d;
}

// f(type, widths): the two sets of widths that are built; others run in the next larger, padded with zeros
template <int N, int R, int V> struct Widths { static constexpr int DN = N, DR = R, DV = V; };
template <typename F>
static int lat_dispatch(const atomic_latent_args* a, F&& f) {
  const bool small = a->dn <= 64 && a->dr <= 32 && a->dv <= 64;
  if (a->dtype == ATOMIC_BF16) return small ? f(bf16(), Widths<64, 32, 64>()) : f(bf16(), Widths<128, 64, 128>());
  return small ? f(float(), Widths<64, 32, 64>()) : f(float(), Widths<128, 64, 128>());
}

// The forward's parts of the keys: doubled while they fill no more than half of the 512
// places, and of eight tiles or more (B2 T517 over S4500, H6: 111 us in one part, 46 in
// eight and their join, when that was made).
static int fwd_parts(const atomic_latent_args* a) {
  const int64_t wgs = (int64_t)a->batch * a->heads * ((a->tq + 127) / 128), tiles = (a->tk + 63) / 64;
  int p = 1;
  while (p < 16 && p * wgs <= 256 && 8 * p <= tiles) p *= 2;
  return p;
}
static size_t fwd_stat_bytes(const atomic_latent_args* a, int parts) {
  return ((size_t)parts * a->batch * a->heads * a->tq * 2 * sizeof(float) + 255) / 256 * 256;
}
constexpr size_t kNoWorkspace = 16;  // what a size function returns where none is needed (0 is a refusal)

// The backward's parts of the keys (dq) and of the queries (dk, dv), and its workspace.
struct BwdPlan {
  int qrows, qparts, kparts;         // rows a workgroup of the dq kernel
  size_t stat, dkp, pq, pkv, ds;     // bytes; ds: the score gradients, 0 where dq computes them again
};
// The backward's: as long as they fit the 256 CUs (one workgroup each) and have four
// tiles or more (fp32 B2 T512 H4, training: 286 us of kernels in one part, 108 in several).
static int parts_for(int64_t wgs, int64_t tiles) {
  int p = 1;
  while (p < 16 && 2 * p * wgs <= 256 && 4 * p <= tiles) p *= 2;
  return p;
}
// Score gradients up to this size are kept between the two kernels (bf16): both of them
// together take 2040 us against 2380 at B2 T8192 H16 and 880 against 1030 at B8 T4096 H6.
// What the size costs is memory only; 4 GB is 1.4 % of the card's.
constexpr int64_t kMostDs = (int64_t)4 << 30;
static BwdPlan bwd_plan(const atomic_latent_args* a) {
  const int64_t bh = (int64_t)a->batch * a->heads, tile = a->dtype == ATOMIC_BF16 ? 64 : 32;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  BwdPlan p;
  const int64_t per = 2 * bh * a->tk;  // bytes a query row; (the product of both stays in 62 bits)
  const bool keep = a->dtype == ATOMIC_BF16 && stat_rows(a->tq) <= kMostDs / per;
  p.ds = keep ? up((size_t)(per * stat_rows(a->tq))) : 0;
  p.qrows = keep ? 256 : 128;
  p.qparts = parts_for(bh * ((a->tq + p.qrows - 1) / p.qrows), (a->tk + tile - 1) / tile);
  p.kparts = parts_for(bh * ((a->tk + 127) / 128), (a->tq + tile - 1) / tile);
  p.stat = up((size_t)bh * stat_rows(a->tq) * 2 * sizeof(float));
  p.dkp = up((size_t)p.kparts * bh * a->tk * a->dr * sizeof(float));
  p.pq = p.qparts > 1 ? up((size_t)p.qparts * bh * a->tq * (a->dn + a->dr) * sizeof(float)) : 0;
  p.pkv = p.kparts > 1 ? up((size_t)p.kparts * bh * a->tk * (a->dn + a->dv) * sizeof(float)) : 0;
  return p;
}

}  // namespace ah

using namespace ah;

extern "C" size_t atomic_latent_fwd_workspace_size(const atomic_latent_args* a) {
  if (lat_check(a) != ATOMIC_OK) return 0;
  const int parts = fwd_parts(a);
  return parts > 1 ? fwd_stat_bytes(a, parts) + (size_t)parts * a->batch * a->heads * a->tq * a->dv * sizeof(float)
                   : kNoWorkspace;
}

extern "C" int atomic_latent_fwd(const atomic_latent_args* a, const void* q, const void* kv, const void* k_pe,
                                 const int32_t* q_lens, const int32_t* kv_lens, void* o, float* lse, void* o_rest,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = lat_check(a)) return rc;
  if (!q || !kv || !k_pe || !o || !lse) return ATOMIC_ERR_NULL;
  if (!aligned16({q, kv, k_pe, o, o_rest})) return ATOMIC_ERR_SHAPE;
  const int parts = fwd_parts(a);
  if (parts > 1) {
    if (!workspace || workspace_bytes < atomic_latent_fwd_workspace_size(a) || !aligned16({workspace}))
      return ATOMIC_ERR_WORKSPACE;
    ws_tag_clobber(workspace, atomic_latent_fwd_workspace_size(a));
  }
  float* pstat = (float*)workspace;
  float* pacc = (float*)((char*)workspace + fwd_stat_bytes(a, parts));
  const hipStream_t st = (hipStream_t)stream;
  Launch L{a->profile, st};
  return lat_dispatch(a, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    T* rest = sizeof(T) == 2 ? (T*)o_rest : nullptr;
    LatDims d = lat_dims(a);
    d.blocks = (d.T + 127) / 128 * parts;
    int rc = L("latent_fwd", [&] {
      hipLaunchKernelGGL((latent_fwd<T, W::DN, W::DR, W::DV>), dim3((unsigned)(d.B * d.H * d.blocks)), dim3(256), 0, st,
                         d, parts, (const T*)q, (const T*)kv, (const T*)k_pe, q_lens, kv_lens, (T*)o, lse, rest, pacc, pstat);
    });
    if (rc || parts == 1) return rc;
    const int64_t n = (int64_t)d.B * d.H * d.T * (d.dv / 4);
    return L("latent_fwd_join", [&] {
      hipLaunchKernelGGL((latent_fwd_join<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, d, parts, pacc,
                         pstat, (T*)o, lse, rest);
    });
  });
}

extern "C" size_t atomic_latent_bwd_workspace_size(const atomic_latent_args* a) {
  if (lat_check(a) != ATOMIC_OK) return 0;
  const BwdPlan p = bwd_plan(a);
  return p.stat + p.dkp + p.pq + p.pkv + p.ds;
}

extern "C" int atomic_latent_bwd(const atomic_latent_args* a, const void* q, const void* kv, const void* k_pe,
                                 const int32_t* q_lens, const int32_t* kv_lens, const void* o, const float* lse,
                                 const void* o_rest, const void* dout, void* dq, void* dkv, void* dk_pe, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (int rc = lat_check(a)) return rc;
  if (!q || !kv || !k_pe || !o || !lse || !dout || !dq || !dkv || !dk_pe) return ATOMIC_ERR_NULL;
  if (!aligned16({q, kv, k_pe, o, o_rest, dout, dq, dkv, dk_pe})) return ATOMIC_ERR_SHAPE;
  if (!workspace || workspace_bytes < atomic_latent_bwd_workspace_size(a) || !aligned16({workspace}))
    return ATOMIC_ERR_WORKSPACE;
  ws_tag_clobber(workspace, atomic_latent_bwd_workspace_size(a));
  const BwdPlan p = bwd_plan(a);
  float* stat = (float*)workspace;
  float* dkp = (float*)((char*)stat + p.stat);
  float* pq = (float*)((char*)dkp + p.dkp);
  float* pkv = (float*)((char*)pq + p.pq);
  void* ds = (char*)pkv + p.pkv;
  const hipStream_t st = (hipStream_t)stream;
  Launch L{a->profile, st};
  return lat_dispatch(a, [&](auto t, auto w) {
    typedef decltype(t) T;
    typedef decltype(w) W;
    LatDims d = lat_dims(a);
    const int64_t rows = (int64_t)d.B * stat_rows(d.T) * d.H;
    int rc = L("latent_delta", [&] {
      hipLaunchKernelGGL((latent_delta<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, d, (const T*)o,
                         sizeof(T) == 2 ? (const T*)o_rest : nullptr, (const T*)dout, lse, q_lens, stat);
    });
    if (rc) return rc;
    d.blocks = (d.S + 127) / 128 * p.kparts;
    rc = L("latent_bwd_dkv", [&] {
      auto go = [&](auto keep) {
        hipLaunchKernelGGL((latent_bwd_dkv<T, W::DN, W::DR, W::DV, decltype(keep)::value != 0>),
                           dim3((unsigned)(d.B * d.H * d.blocks)), dim3(256), 0, st, d, (const T*)q, (const T*)kv,
                           (const T*)k_pe, q_lens, kv_lens, stat, (const T*)dout, (T*)dkv, dkp, p.kparts, pkv,
                           (T*)ds);
      };
      if constexpr (sizeof(T) == 2) {
        if (p.ds) go(IntC<1>());
        else go(IntC<0>());
      } else {
        go(IntC<0>());
      }
    });
    if (rc) return rc;
    d.blocks = (d.T + p.qrows - 1) / p.qrows * p.qparts;
    rc = L("latent_bwd_dq", [&] {
      const dim3 grid((unsigned)(d.B * d.H * d.blocks));
      if constexpr (sizeof(T) == 2) {
        if (p.ds) {
          hipLaunchKernelGGL((latent_bwd_dq_ds<W::DN, W::DR>), grid, dim3(256), 0, st, d, (const T*)kv,
                             (const T*)k_pe, q_lens, kv_lens, (const T*)ds, (T*)dq, p.qparts, pq);
          return;
        }
      }
      hipLaunchKernelGGL((latent_bwd_dq<T, W::DN, W::DR, W::DV>), grid, dim3(256), 0, st, d, (const T*)q,
                         (const T*)kv, (const T*)k_pe, q_lens, kv_lens, stat, (const T*)dout, (T*)dq, p.qparts, pq);
    });
    if (rc) return rc;
    FinishJobs f{p.kparts > 1 ? (int64_t)d.B * d.S * d.H * (d.dn + d.dv) : 0,
                 p.qparts > 1 ? (int64_t)d.B * d.T * d.H * (d.dn + d.dr) : 0, 0, 0, p.kparts, p.qparts};
    f.b1 = (unsigned)((f.n1 / 4 + 255) / 256);
    f.b2 = (unsigned)((f.n2 / 4 + 255) / 256);
    const unsigned b3 = (unsigned)(((int64_t)d.B * d.S * d.dr / 4 + 255) / 256);
    return L("latent_bwd_finish", [&] {
      hipLaunchKernelGGL((latent_bwd_finish<T>), dim3(f.b1 + f.b2 + b3), dim3(256), 0, st, d, f, pkv, pq, dkp,
                         (T*)dkv, (T*)dq, (T*)dk_pe);
    });
  });
}
