// The absorbed form over a prefix that many query rows share, for gfx950: with 64
// sequences of 16 heads a prefix token is read once for 1024 rows, so that matrix
// instructions bound it (1900 operations a byte), not the cache's bytes.
#include "latent_decode.hpp"

#ifndef XG
#define XG 2
#define XL 2
#endif
#ifndef YG
#define YG 2
#define YL 2
#endif
#ifndef YV
#define YV 4
#endif
namespace ah {

// Keep a value in the accumulator half of the register file.
template <typename F> __device__ __forceinline__ void in_accum(F& x) { asm volatile("" : "+a"(x)); }

// x *= f for an x there.  (Written as a product, the compiler reads all accumulators ahead of the
// branch that this is in, into registers that are not there.)
__device__ __forceinline__ void accum_mul(float& x, float f) {
  float y;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(x), "=&v"(y)
               : "v"(f));
}

constexpr int kPreRows = 128, kPreTokens = 32, kPreBufs = 4, kPreChunk = 2048;

template <int DC>
__global__ __launch_bounds__(256, 1) void latent_prefix(DecDims d, int blocks, int units,
                                                        const bf16* __restrict__ qa, const bf16* __restrict__ cache,
                                                        const int32_t* __restrict__ table,
                                                        const int32_t* __restrict__ lens,
                                                        const int32_t* __restrict__ own, int own_most,
                                                        float* __restrict__ part, float* __restrict__ stat) {
  constexpr int DR = 64, KS = (DC + DR) / 16, KC = DC / 16, NT = DC / 32, TK = kPreTokens;
  typedef LTile<bf16, DC> LC;
  typedef LTile<bf16, DR> LR;
  typedef bf16x8 frag;
  constexpr int SC = TK * LC::ROWB, SR = TK * LR::ROWB, STAGE = SC + SR;
  constexpr int PT = TK / 4, NL = PT + 1;  // a wave's tokens of a tile, and its loads
  static_assert(DC == 512, "a latent is one load of a wave");
  __shared__ __attribute__((aligned(1024))) char lds[kPreBufs * STAGE];
  __shared__ uint32_t slot[kPreChunk];
  // the row blocks of a split on one XCD, whose L2 then holds the split's tokens
  int sp, blk;
  xcd_group_map(blockIdx.x, d.splits * units, blocks, sp, blk);
  const int b = sp / d.splits, wv = wave_id(), lane = lane_id();
  sp %= d.splits;
  const int len = dec_len(d, lens, b), each = d.n * d.H, rows = d.share * each, wide = d.dc + d.dr;
  const int first = sp * d.chunk, end = min(len, first + d.chunk);
  if (first >= end) return;
  for (int i = threadIdx.x; i < end - first; i += 256) {
    const int j = first + i, pg = j / d.page;
    slot[i] = (uint32_t)min(max(table[(int64_t)b * d.table + pg], 0), d.pages - 1) * d.page + (j - pg * d.page);
  }
  const int row = kPreRows * blk + 32 * wv + (lane & 31), at = min(row, rows - 1);
  const int seq = b * d.share + at / each, place = at % each;
  const int seen = len + min(max(own[seq], 0), own_most) - d.n + place / d.H + 1;  // tokens that this lane's row sees
  const int least = len - d.n + 1;                                                 // and that every row sees
  const bf16* qr = qa + ((int64_t)seq * each + place) * wide;
  frag qf[KS];
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    const int k = 16 * t + 8 * (lane >> 5);
    if (t < KC) qf[t] = ld_frag(k < d.dc ? qr + k : (const bf16*)lat_zeros);
    else qf[t] = ld_frag(k - DC < d.dr ? qr + d.dc + k - DC : (const bf16*)lat_zeros);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  __syncthreads();  // the rows' places are there
  const uint32_t l0 = lds_addr(lds), wb = 2 * d.dc;
  // This wave's loads of the tile at k0 (from `first` on): eight latents, then their rotated keys.
  uint32_t lo, hi;
  auto aim = [&](int k0) {
    const uint64_t a = (uint64_t)cache + (uint64_t)slot[min(k0 + PT * wv + (lane & 7), end - first - 1)] * (2 * wide);
    lo = (uint32_t)a;
    hi = (uint32_t)(a >> 32);
  };
  auto load = [&](int i, uint32_t to) {
    if (i < PT) {
      const int r = PT * wv + i;
      const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, i) << 32 |
                            (uint32_t)__builtin_amdgcn_readlane(lo, i);
      uint32_t off = 16 * lane ^ 16 * LC::swz(r);
      if (off >= wb) off = 0;  // the padding of a width: the query has zeros there
      dma16_raw_s(base, off, to + r * LC::ROWB);
    } else {
      const int r = PT * wv + lane / 8;
      const uint64_t base = (uint64_t)__shfl(hi, lane / 8) << 32 | (uint32_t)__shfl(lo, lane / 8);
      uint32_t off = 16 * (lane % 8) ^ 16 * LR::swz(r);
      if (off >= 2 * (uint32_t)d.dr) off = 0;
      dma16_raw((const void*)(base + wb + off), to + SC + PT * wv * LR::ROWB);
    }
  };
  f32x16 acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = zero16();
  // (a scale of zero as the smallest number: a masked score stays infinite; a negative one changes q's sign)
  const float c2 = d.scale == 0.f ? 1.17549435e-38f : fabsf(d.scale) * kLog2e;
  if (d.scale < 0.f) {
#pragma unroll
    for (int t = 0; t < KS; ++t) qf[t] = -qf[t];
  }
  float m = -INFINITY, sum = 0.f;
  f32x16 s;
  const uint32_t br = LC::row_base(), bp = LR::row_base(), bc = LC::col_base();
  // Scores of the tile at k0, masked.
  auto scores = [&](int buf, int k0, auto work) {
    uint32_t ac = l0 + buf * STAGE + br, ar = l0 + buf * STAGE + SC + bp;
    asm volatile("" : "+v"(ac), "+v"(ar));
    s = zero16();
#ifdef CH2
    f32x16 s1 = zero16();
#endif
    in_groups<KS, XG, XL, 0, frag>([&](int t) { return t < KC ? LC::row(ac, 0, 16 * t) : LR::row(ar, 0, 16 * (t - KC)); },
                                 [&](int t, frag a) {
#ifdef CH2
                                   if (t & 1) s1 = M32<bf16>::mma(a, qf[t], s1);
                                   else
#endif
                                   s = M32<bf16>::mma(a, qf[t], s); }, work);
#ifdef CH2
    s += s1;
#endif
    asm volatile("" : "+v"(s));
    if (first + k0 + TK > min(end, least)) {
      const int lim = min(end, seen) - first - k0 - 4 * (lane >> 5);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        int z = lim;
        asm volatile("" : "+v"(z));
        s[r] = 8 * (r >> 2) + (r & 3) < z ? s[r] : -INFINITY;
      }
    }
  };
  frag p[2], pn[2];
  auto quad = [&](int k) {  // four tokens' probabilities
    const float ref = m == -INFINITY ? 0.f : -m;  // a row that has seen nothing yet: every p is exp2(-inf) = 0
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float e = fast_exp2(__builtin_fmaf(s[4 * k + j], c2, ref));
      sum += e;
      pn[k / 2][4 * (k & 1) + j] = (bf16)e;
    }
  };
  // A tile's probabilities times its latents; beside them `work`.
  auto values = [&](int buf, auto work) {
    uint32_t av = l0 + buf * STAGE + bc;
    asm volatile("" : "+v"(av));
    in_groups<2 * NT, YG, YL, YV, frag>([&](int j) { return LC::col(av, 16 * (j / NT), 32 * (j % NT)); },
                                     [&](int j, frag a) { acc[j % NT] = M32<bf16>::mma(a, p[j / NT], acc[j % NT]); },
                                     work);
#pragma unroll
    for (int n = 0; n < NT; ++n) in_accum(acc[n]);
  };
  // A new reference where a score is far above its row's: a whole number, so that what
  // fades, the last tile's probabilities among it, is scaled exactly.
  auto settle = [&] {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top *= c2;
    if (__any(top > m + kLag)) {
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, ceilf(top)), fade = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
      m = mn;
      sum *= fade;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) p[k][j] = (bf16)((float)p[k][j] * fade);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float z = acc[n][r];
          accum_mul(z, fade);
          acc[n][r] = z;
        }
      }
      asm volatile("s_nop 7" ::: "memory");
    }
  };
  const int tiles = (end - first + TK - 1) / TK;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    aim(TK * k);
#pragma unroll
    for (int i = 0; i < NL; ++i) load(i, l0 + k * STAGE);
  }
  vm_wait<2 * NL>();
  bare_barrier();
  p[0] = p[1] = zero_frag<bf16>();
  scores(0, 0, [](int) {});
  settle();
#pragma unroll
  for (int k = 0; k < 4; ++k) quad(k);
  p[0] = pn[0];
  p[1] = pn[1];
  for (int i = 1; i < tiles; ++i) {
    vm_wait<NL>();   // tile i is there (of this wave's loads; behind the barrier, of all)
    bare_barrier();  // and nobody reads tile i - 2 any more
    aim(TK * (i + 2));
    const uint32_t to = l0 + (i + 2) % kPreBufs * STAGE;
    scores(i % kPreBufs, TK * i, [&](int t) {
#pragma unroll
      for (int j = 0; j < NL; ++j)
        if (j * KS / NL == t) load(j, to);
    });
    settle();
    values((i - 1) % kPreBufs, [&](int j) {
      if (j % 8 == 2) quad(j / 8);
    });
    p[0] = pn[0];
    p[1] = pn[1];
  }
  values((tiles - 1) % kPreBufs, [](int) {});
  vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
  if (row >= rows) return;
  sum += __shfl_xor(sum, 32);
  const int64_t to = ((int64_t)seq * d.slots + d.slot0 + sp) * each + place;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int c = 32 * n + 8 * (r >> 2) + 4 * (lane >> 5);
      if (c < d.dc) store4(part + to * d.dc + c, f32x4{acc[n][r], acc[n][r + 1], acc[n][r + 2], acc[n][r + 3]});
    }
  if (lane < 32) {
    stat[2 * to] = m;
    stat[2 * to + 1] = sum;
  }
}

bool prefix_plan(DecDims& d, int units) {
  const int64_t rows = (int64_t)d.share * d.n * d.H, most = (int64_t)d.table * d.page;
  if (rows <= 32 || most < 256 || (int64_t)d.pages * d.page > UINT32_MAX) return false;
  const int64_t blocks = (rows + kPreRows - 1) / kPreRows * units;
  double best = 0;
  for (int chunk = 64; chunk <= kPreChunk; chunk += 32) {
    const int64_t wg = blocks * ((most + chunk - 1) / chunk);
    const double cost = (double)((wg + 255) / 256) * (0.034 * chunk + 4) + 0.13 * (double)wg;
    if (chunk == 64 || cost < best) {
      best = cost;
      d.chunk = chunk;
    }
  }
  d.splits = (int)((most + d.chunk - 1) / d.chunk);
  return blocks * d.splits <= INT32_MAX;
}

void launch_prefix(const DecDims& d, int units, hipStream_t st, const bf16* qa, const void* cache, const int32_t* table,
                   const int32_t* lens, const int32_t* own, int own_most, float* part, float* stat) {
  const int blocks = (int)(((int64_t)d.share * d.n * d.H + kPreRows - 1) / kPreRows);
  hipLaunchKernelGGL((latent_prefix<512>), dim3((unsigned)(d.splits * units * blocks)), dim3(256), 0, st, d, blocks,
                     units, qa, (const bf16*)cache, table, lens, own, own_most, part, stat);
}

}  // namespace ah
