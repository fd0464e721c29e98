// The absorbed form over a prefix that many query rows share, for gfx950: with 64
// sequences of 16 heads a prefix token is read once for 1024 rows, so that matrix
// instructions bound it (1900 operations a byte), not the cache's bytes.
//
// A workgroup takes 128 rows, 32 a wave, and a split of the prefix in tiles of 32 tokens:
//   s = K q^T      tokens x rows: a lane holds 16 tokens' scores of its row
//   p = 2^(s - m)  in registers, which are the B operand of the next product as they stand
//   o^T += C^T p   latents x rows, in the accumulator half of the register file
// Each MFMA reads 1 KB of LDS, so a tile costs a wave 36 + 32 of them (and 4 for the rest of
// the rotated queries) and as many reads; all four waves read the same tile, four tiles are
// in LDS, and loads, reads and MFMAs are spread over each other by hand (`tile`).  The scores of
// tile i and the products of tile i - 1 are one run, so that the softmax of one lies under
// the products of the other.  A tile takes 4000 clocks (2.2 us), 2304 of them its 72
// MFMAs.  64 sequences of 16 heads over 32768 tokens and their 512 own ones: 97 us, 0.77
// PFLOP/s (latent_split took 150 for the prefix alone); over 8192 and up to 1024: 47 us.  What is
// not tiles, 38 % of the clocks of the first, is the queries, which have to be there before the first
// product (128 KB a workgroup), the parts (67 MB there) and the own tokens.  More operands
// read ahead, two chains of scores and, with 256 latents, seven tiles in LDS changed nothing.
//
// From 2048 tokens of a prefix on p enters as one bf16 number: o is off by 0.0025 of its norm
// behind 2048 to 4096 of them and 0.0024 behind 8192, where latent_split, which has two, is at
// 0.0023 to 0.0024 and o's own rounding at 0.0017 (the rest is q_lat's).  Behind 64 to 1024 it
// was 0.0025 to 0.0027; there p is two numbers here too, whatever the table's width, and o off
// by 0.0022 (with one, 32 of 104 MFMAs a tile less: four prefixes of 2049 to 4096 tokens, 512
// rows each, 61 us a call, and 68 with two).
#include "latent_decode.hpp"

namespace ah {

// x *= f for an x there.  (Written as a product, the compiler reads all accumulators ahead of the
// branch that this is in, into registers that are not there.)
__device__ __forceinline__ void accum_mul(float& x, float f) {
  float y;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(x), "=&v"(y)
               : "v"(f));
}

constexpr int kPreRows = 128, kPreTokens = 32, kPreBufs = 4, kPreChunk = 2048;
constexpr int kPreOne = 2048;  // tokens of a prefix from which on p enters as one bf16 number
constexpr int kPreTable = 4096;  // tokens that a prefix's table has at least
static_assert(kPreTable >= 2 * kPreChunk, "two splits or more: a row's parts are always joined");

template <int DC> struct PrefixLds {
  // (seven tiles of 256 latents, for which there is room, were no faster)
  char lds[kPreBufs * kPreTokens * (LTile<bf16, DC>::ROWB + LTile<bf16, 64>::ROWB)];
  uint32_t slot[kPreChunk];
};
// The address that lane r holds, and those of lanes r and r + 1 in the lower and upper half of a wave.
__device__ __forceinline__ uint64_t row_at(uint32_t lo, uint32_t hi, int r) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, r) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, r);
}
__device__ __forceinline__ uint64_t pair_at(uint32_t lo, uint32_t hi, int r) {
  return lane_id() < 32 ? row_at(lo, hi, r) : row_at(lo, hi, r + 1);
}
// What lane r holds.  (__shfl keeps two registers more.)
template <typename X> __device__ __forceinline__ X lane_at(X x, int r) {
  return __builtin_bit_cast(X, __builtin_amdgcn_ds_bpermute(4 * r, __builtin_bit_cast(int, x)));
}
// Workgroup `id` of those over the prefixes.
//
// p enters its products as one bf16 number, so a row's average of the latents is theirs by the
// sum of those numbers, `held`.  (By the sum of p itself a row that looks at one token was off
// by that one's rounding, up to 2^-8.)  Where the tokens' weights are gathered the row's sum has to
// be that of p, and the products are scaled to it.
template <int DC, bool SCORED>
__device__ __forceinline__ void prefix_tokens(const DecDims& d, PrefixLds<DC>& mem, int id, int blocks, int units,
                                              const bf16* __restrict__ qa, const bf16* __restrict__ cache,
                                              const int32_t* __restrict__ table, const int32_t* __restrict__ lens,
                                              const int32_t* __restrict__ own, int own_most, f32x4* __restrict__ parts,
                                              float* __restrict__ stat) {
  constexpr int DR = 64, KS = (DC + DR) / 16, KC = DC / 16, NT = DC / 32, TK = kPreTokens;
  typedef LTile<bf16, DC> LC;
  typedef LTile<bf16, DR> LR;
  typedef bf16x8 frag;
  constexpr int SC = TK * LC::ROWB, SR = TK * LR::ROWB, STAGE = SC + SR;
  constexpr int PL = DC / 8, RL = 64 / PL;      // lanes that load a latent, latents of a load
  constexpr int NB = kPreBufs;
  constexpr int PT = TK / 4, NL = PT / RL + 1;  // a wave's tokens of a tile, and its loads
  static_assert(DC == 512 || DC == 256, "a latent, or two, are one load of a wave");
  uint32_t* const slot = mem.slot;
  // the row blocks of a split on one XCD, whose L2 then holds the split's tokens
  int sp, blk;
  xcd_group_map(id, d.splits * units, blocks, sp, blk);
  const int b = sp / d.splits, wv = wave_id(), lane = lane_id();
  const int pl = RL == 1 ? lane : lane % PL, lr = RL == 1 ? 0 : lane / PL;  // this lane's piece and latent of a load
  sp %= d.splits;
  const int each = d.n * d.H, rows = d.share * each, wide = d.dc + d.dr;
  const int row = kPreRows * blk + 32 * wv + (lane & 31), at = min(row, rows - 1);
  const int seq = b * d.share + at / each, place = at % each;
  // The queries of a wave go through the tile buffer of its number, row by row, while the
  // tokens' places are looked up.  (Loaded as fragments, 32 rows an instruction, they took
  // 9300 clocks.)
  const uint32_t l0 = lds_addr(mem.lds), wb = 2 * d.dc, rb = 2 * d.dr;
  {
    const uint64_t a = (uint64_t)(qa + ((int64_t)seq * each + place) * 2 * wide);
    const uint32_t lo = (uint32_t)a, hi = (uint32_t)(a >> 32), to = l0 + wv * STAGE;
#pragma unroll
    for (int i = 0; i < 32 / RL; ++i) {
      const int r = RL * i + lr;
      const uint64_t base = RL == 1 ? row_at(lo, hi, i) : pair_at(lo, hi, 2 * i);
      const uint32_t off = 16 * pl ^ 16 * LC::swz(r);
      dma16_raw((const void*)(off < wb ? base + off : (uint64_t)lat_zeros), to + RL * i * LC::ROWB);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + lane / 8;
      const uint64_t base = (uint64_t)lane_at(hi, r) << 32 | lane_at(lo, r);
      const uint32_t off = 16 * (lane % 8) ^ 16 * LR::swz(r);
      dma16_raw((const void*)(off < rb ? base + wb + off : (uint64_t)lat_zeros), to + SC + 8 * i * LR::ROWB);
    }
  }
  const int len = dec_len(d, lens, b);
  const int first = sp * d.chunk, end = min(len, first + d.chunk);
  if (first >= end) {
    vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
    return;
  }
  for (int i = threadIdx.x; i < end - first; i += 256) {
    const int j = first + i, pg = j / d.page;
    slot[i] = (uint32_t)min(max(table[(int64_t)b * d.table + pg], 0), d.pages - 1) * d.page + (j - pg * d.page);
  }
  const int seen = len + min(max(own[seq], 0), own_most) - d.n + place / d.H + 1;  // tokens that this lane's row sees
  const int least = len - d.n + 1;                                                 // and that every row sees
  vm_wait<0>();
  frag qf[KS];
  {
    const uint32_t ac = l0 + wv * STAGE + LC::row_base(), ar = l0 + wv * STAGE + SC + LR::row_base();
#pragma unroll
    for (int t = 0; t < KS; ++t) qf[t] = t < KC ? LC::row(ac, 0, 16 * t) : LR::row(ar, 0, 16 * (t - KC));
  }
  // What the rounding of the rotated queries left out enters the scores too.
  frag ql[KS - KC];
  {
    const bf16* qr = qa + (((int64_t)seq * each + place) * 2 + 1) * wide + d.dc;
#pragma unroll
    for (int t = 0; t < KS - KC; ++t) {
      const int k = 16 * t + 8 * (lane >> 5);
      ql[t] = ld_frag(k < d.dr ? qr + k : (const bf16*)lat_zeros);
    }
  }
  __syncthreads();  // the tokens' places are there, the buffers free
  // This wave's loads of the tile at k0 (from `first` on): eight latents, then their rotated keys.
  // (Their places are read a tile ahead.)
  uint32_t lo, hi, next, off0;  // (off0: each load's offset from it when it is sent, not eight of them kept over the tiles)
  auto look = [&](int k0) { next = slot[min(k0 + PT * wv + (lane & 7), end - first - 1)]; };
  auto aim = [&] {
    const uint64_t a = (uint64_t)cache + (uint64_t)next * (2 * wide);
    lo = (uint32_t)a;
    hi = (uint32_t)(a >> 32);
    off0 = 16 * pl;
    asm volatile("" : "+v"(off0));
  };
  auto send = [&](int i, uint32_t to) __attribute__((always_inline)) {
    if (i < PT / RL) {
      const int r = PT * wv + RL * i;
      uint32_t off = off0 ^ 16 * LC::swz(r + lr);
      if (off >= wb) off = 0;  // the padding of a width: the query has zeros there
      if constexpr (RL == 1) dma16_raw_s(row_at(lo, hi, i), off, to + r * LC::ROWB);
      else dma16_raw((const void*)(pair_at(lo, hi, 2 * i) + off), to + r * LC::ROWB);
    } else {
      int ln = lane;
      asm volatile("" : "+v"(ln));
      const int r = PT * wv + ln / 8;
      const uint64_t base = (uint64_t)lane_at(hi, ln / 8) << 32 | lane_at(lo, ln / 8);
      uint32_t off = 16 * (ln % 8) ^ 16 * LR::swz(r);
      if (off >= rb) off = 0;
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
#pragma unroll
    for (int t = 0; t < KS - KC; ++t) ql[t] = -ql[t];
  }
  float m = -INFINITY, sum = 0.f, held = 0.f;
  f32x16 s;
  const uint32_t br = LC::row_base(), bp = LR::row_base(), bc = LC::col_base();
  auto mask = [&](int k0) __attribute__((always_inline)) {
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
  typedef bf16 pair __attribute__((ext_vector_type(2)));
  // All tiles, with p as NP bf16 numbers.
  auto walk = [&](auto numbers) __attribute__((always_inline)) {
    constexpr int NP = decltype(numbers)::value;
    frag p[2], pn[NP][2];  // the last tile's, and this one's
    auto quad = [&](int k) __attribute__((always_inline)) {  // four tokens' probabilities
      const float ref = m == -INFINITY ? 0.f : -m;  // a row that has seen nothing yet: every p is exp2(-inf) = 0
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float e = fast_exp2(__builtin_fmaf(s[4 * k + j], c2, ref));
        if constexpr (SCORED) sum += e;
#pragma unroll
        for (int u = 0; u < NP; ++u) {
          const bf16 h = (bf16)e;
          pn[u][k / 2][4 * (k & 1) + j] = h;
          e -= (float)h;
        }
      }
      const pair one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
      for (int u = 0; u < NP; ++u)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const int at = 4 * (k & 1) + j;
          held = __builtin_amdgcn_fdot2_f32_bf16(pair{pn[u][k / 2][at], pn[u][k / 2][at + 1]}, one, held, false);
        }
    };
    // A new reference where a score is far above its row's: a whole number, so that what
    // fades, the last tile's probabilities among it, is scaled exactly.
    auto settle = [&](auto fades) __attribute__((always_inline)) {
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      top *= c2;
      if (__any(top > m + kLag)) {
        top = fmaxf(top, lane_at(top, lane ^ 32));
        const float mn = fmaxf(m, ceilf(top)), fade = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
        m = mn;
        if constexpr (!decltype(fades)::value) return;  // (the first tile: nothing is there yet)
        if constexpr (SCORED) sum *= fade;
        held *= fade;
        if constexpr (NP == 1) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) p[k][j] = (bf16)((float)p[k][j] * fade);
        }
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
    // The scores of tile i in buffer `kb` and the products of the tile before in `vb`, as one run
    // of groups of G MFMAs whose operands are read LA groups ahead, so that the second part
    // does not begin with a wait.  Either part may be left out (`kb`, `vb` below zero).
    constexpr int G = 1, LA = 2, GS = KS / G, GV = 2 * NT / G;
    auto tile = [&](auto with_k, auto with_v, auto sends, int kb, int vb, int k0, uint32_t to) __attribute__((always_inline)) {
      constexpr int g0 = decltype(with_k)::value ? 0 : GS, g1 = decltype(with_v)::value ? GS + GV : GS;
      uint32_t ac = l0 + kb * STAGE + br, ar = l0 + kb * STAGE + SC + bp, av = l0 + vb * STAGE + bc;
      asm volatile("" : "+v"(ac), "+v"(ar), "+v"(av));
      auto load = [&](int j) {
        return j < KC ? LC::row(ac, 0, 16 * j)
                      : j < KS ? LR::row(ar, 0, 16 * (j - KC)) : LC::col(av, 16 * ((j - KS) / NT), 32 * ((j - KS) % NT));
      };
      frag f[LA + 1][G];
      static_for<LA * G>([&](auto j) { f[(g0 + j.value / G) % (LA + 1)][j.value % G] = load(g0 * G + j.value); });
      __builtin_amdgcn_sched_barrier(0);
      static_for<g1 - g0>([&](auto gr) __attribute__((always_inline)) {
        constexpr int g = g0 + decltype(gr)::value;
        static_for<G>([&](auto j) {
          if constexpr (g + LA < g1) f[(g + LA) % (LA + 1)][j.value] = load((g + LA) * G + j.value);
        });
        if constexpr (g < GS) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int j = 0; j < NL; ++j)
            if (decltype(sends)::value && j * GS / NL == g) send(j, to);
          if constexpr (g == 0) s = zero16();
          static_for<G>([&](auto j) {
            constexpr int t = g * G + decltype(j)::value;
            s = M32<bf16>::mma(f[g % (LA + 1)][j.value], qf[t], s);
            if constexpr (t >= KC) s = M32<bf16>::mma(f[g % (LA + 1)][j.value], ql[t - KC], s);
          });
          if constexpr (g == GS - 1) {
            asm volatile("" : "+v"(s));
            mask(k0);
            settle(sends);  // (the first tile sends no other)
          }
        } else {
          if constexpr (decltype(with_k)::value && (g - GS) % (GV / 4) == 1) quad((g - GS) / (GV / 4));
          static_for<G>([&](auto j) {
            constexpr int v = (g - GS) * G + decltype(j)::value;
            if constexpr (NP == 1) acc[v % NT] = M32<bf16>::mma(f[g % (LA + 1)][j.value], p[v / NT], acc[v % NT]);
            else
#pragma unroll
              for (int u = 0; u < NP; ++u) acc[v % NT] = M32<bf16>::mma(f[g % (LA + 1)][j.value], pn[u][v / NT], acc[v % NT]);
          });
          __builtin_amdgcn_sched_group_barrier(0x100, 4 * G, 0);  // LDS reads
          static_for<NP * G>([&](auto) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // vector
          });
        }
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (decltype(with_v)::value) {
#pragma unroll
        for (int n = 0; n < NT; ++n) in_accum(acc[n]);
      }
    };
    const int tiles = (end - first + TK - 1) / TK;
#pragma unroll
    for (int k = 0; k < NB - 1; ++k) {
      look(TK * k);
      aim();
#pragma unroll
      for (int i = 0; i < NL; ++i) send(i, l0 + k * STAGE);
    }
    look(TK * (NB - 1));
    vm_wait<(NB - 2) * NL>();
    bare_barrier();
    const IntC<0> no;
    const IntC<1> yes;
    tile(yes, no, no, 0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 4; ++k) quad(k);
    if constexpr (NP == 1) {
      p[0] = pn[0][0];
      p[1] = pn[0][1];
    } else {
      tile(no, yes, no, 0, 0, 0, 0);
    }
    for (int i = 1; i < tiles; ++i) {
      vm_wait<(NB - 3) * NL>();  // tile i is there (of this wave's loads; behind the barrier, of all)
      bare_barrier();            // and nobody reads tile i - 2 any more
      aim();
      look(TK * (i + NB - 1));
      const uint32_t to = l0 + (i + NB - 2) % NB * STAGE;
      if constexpr (NP == 1) {
        tile(yes, yes, yes, i % NB, (i - 1) % NB, TK * i, to);
        p[0] = pn[0][0];
        p[1] = pn[0][1];
      } else {  // (the products of the same tile: two numbers of two tiles would be 16 registers more)
        tile(yes, no, yes, i % NB, 0, TK * i, to);
#pragma unroll
        for (int k = 0; k < 4; ++k) quad(k);
        tile(no, yes, no, 0, i % NB, 0, 0);
      }
    }
    if constexpr (NP == 1) tile(no, yes, no, 0, (tiles - 1) % NB, 0, 0);
  };
  if (len < kPreOne) walk(IntC<2>());
  else walk(IntC<1>());
  vm_wait<0>();  // nothing is on its way to LDS when the workgroup ends
  held += lane_at(held, lane ^ 32);
  if constexpr (SCORED) sum += lane_at(sum, lane ^ 32);
  else sum = held;
  const float even = SCORED && held != 0.f ? sum / held : 1.f;
  // A part: a lane's accumulators four by four, in the order that they have.
  const int64_t group = ((int64_t)b * blocks + blk) * 4 + wv;
  // (this lane and its row once more, so that they are not kept over the tiles)
  const int row0 = kPreRows * blk + 32 * wv + opaque_zero();
  const int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, opaque_zero()));
  f32x4* to = parts + (group * d.splits + sp) * (4 * NT * 64) + ln;
  const int columns = kPreRows * blk + 32 * wv < rows ? d.dc : 0;  // (nobody reads a part without rows)
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f32x4 x = {acc[n][4 * k], acc[n][4 * k + 1], acc[n][4 * k + 2], acc[n][4 * k + 3]};
      if constexpr (SCORED) x *= even;
      if (32 * n < columns) to[(4 * n + k) * 64] = x;
    }
  if (ln < 32 && row0 + ln < rows) {
    const int of = each + opaque_zero(), own_seq = b * d.share + (row0 + ln) / of;
    const int64_t at = ((int64_t)own_seq * d.slots + d.slot0 + sp) * of + (row0 + ln) % of;
    stat[2 * at] = m;
    stat[2 * at + 1] = sum;
  }
}

// Both kinds of workgroups in one launch: those over the prefixes and, on the CUs that they
// leave and behind them, those over the own tokens.  Where there is a prefix workgroup for every CU,
// `early` of the others, up to half a card of them, go first: half of the CUs then begin with
// the one kind and end with the other.  What is bound by memory so runs beside what is bound by
// matrix instructions (64 sequences of 16 heads over 8192 tokens and up to 1024 own
// ones, 47 us.  Whole calls, measured with parts of half the bytes: 32 sequences over 8192 and 2048 tokens with
// weights 77 us in two launches and 71 in one; 64 over 32768 and 512 132 with the two kinds by turns and 109 so).
template <int DC, int MT, bool SCORED>
__global__ __launch_bounds__(256, 1) void latent_prefix(PrefixCall c, int blocks, int early, f32x4* __restrict__ parts) {
  typedef SplitLds<bf16, DC, 4> OwnLds;
  typedef PrefixLds<DC> PreLds;
  __shared__ __attribute__((aligned(1024))) char mem[sizeof(PreLds) > sizeof(OwnLds) ? sizeof(PreLds) : sizeof(OwnLds)];
  const DecDims& d = c.d;
  const int front = c.f.splits * c.units * blocks, at = (int)blockIdx.x - early;
  if (at >= 0 && at < front) {
    prefix_tokens<DC, SCORED>(c.f, *reinterpret_cast<PreLds*>(mem), at, blocks, c.units, c.qa, c.cache, c.prefix_table,
                       c.prefix_lens, c.lens, d.table * d.page, parts, c.stat);
  } else {
    const int id = at < 0 ? (int)blockIdx.x : (int)blockIdx.x - front;
    split_tokens<bf16, DC, MT, 4, SCORED, false>(d, *reinterpret_cast<OwnLds*>(mem), id % d.splits, id / d.splits % d.groups,
                                           id / d.splits / d.groups, c.qa, c.cache, c.table, c.lens, nullptr, 0, c.part,
                                           c.stat, c.olat, c.score);
  }
}

// o_lat of the rows behind a prefix: latent_prefix's parts and those of the sequences' own
// tokens joined.  A workgroup takes 32 rows and 64 (or 16) columns, eight (two) of the parts'
// blocks of 1 KB; a wave has two of them and every WAYS-th split.
//
// Where the tokens' weights are gathered, `shift` [rows, 8] receives what q_lat's rounding did
// to the log (base 2) of a row's sum over the prefix: with e = q_lat - its bf16, a score is off
// by c e . c_j, so the log by c e . (sum_j p_j c_j) and, what is left, half the variance of
// c e . c_j, which grows with the scores: gathered weights are off by 1.5e-6 of their norm where
// scores have unit spread, 9e-6 at a spread of 3 and 2e-5 to 3e-5 at 10; with the second number in every
// score, as latent_split has it, by 1e-6, 4e-6 and 8e-6.  (Uncorrected 5e-5 at unit spread.)
// Each workgroup gives its 64 columns' share.  (As a second number in the scores it would
// take another 32 of 36 matrix instructions a tile and 128 registers that are not there.)
template <int DC, int COLS, int WAYS>
__global__ __launch_bounds__(4 * COLS * WAYS) void latent_prefix_join(DecDims f, DecDims d, int blocks, const f32x4* __restrict__ parts,
                                                          const float* __restrict__ part,
                                                          const float* __restrict__ stat,
                                                          const int32_t* __restrict__ kv_lens,
                                                          float* __restrict__ olat, const bf16* __restrict__ qa,
                                                          float* __restrict__ shift) {
  constexpr int NT = DC / 32, CB = DC / COLS, NB = COLS / 16, LD = COLS + 4;
  __shared__ float ms[WAYS][32], ss[WAYS][32];
  __shared__ __attribute__((aligned(16))) float tile[WAYS][32 * LD];
  const int group = blockIdx.x / CB, cb = blockIdx.x % CB, k = NB * cb + wave_id() % NB, way = wave_id() / NB, lane = lane_id();
  const int each = d.n * d.H, rows = f.share * each, b = group / (4 * blocks), r0 = 32 * (group % (4 * blocks));
  if (r0 >= rows) return;
  // Both kinds of parts with a reference of their own, so that nothing waits for the other's
  // statistics: the prefix's, a row a lane,
  {
    const int row = min(r0 + (lane & 31), rows - 1), seq = b * f.share + row / each, place = row % each;
    const int n = Parts<true>(d, kv_lens, seq).front;
    const float* st = stat + 2 * ((int64_t)seq * d.slots * each + place);
    const f32x4* from = parts + (int64_t)group * f.splits * (4 * NT * 64) + (32 * (k / 2) < d.dc ? k : 0) * 128 + lane;
    f32x4 x[2] = {zero4(), zero4()};
    float m = -INFINITY, sum = 0.f;
    for (int s0 = way; s0 < n; s0 += 8 * WAYS) {
      f32x4 y[8][2];
      float2 a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // (splits past the last repeat it, with a weight of zero)
        const int s = min(s0 + WAYS * i, n - 1);
        a[i] = *reinterpret_cast<const float2*>(st + 2 * (int64_t)s * each);
        y[i][0] = from[(int64_t)s * (4 * NT * 64)];
        y[i][1] = from[(int64_t)s * (4 * NT * 64) + 64];
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) mn = fmaxf(mn, s0 + WAYS * i < n ? a[i].x : -INFINITY);
      const float ref = mn == -INFINITY ? 0.f : mn, fade = fast_exp2(m - ref);
      m = mn;
      sum *= fade;
      x[0] *= fade;
      x[1] *= fade;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = s0 + WAYS * i < n ? fast_exp2(a[i].x - ref) : 0.f;
        sum += w * a[i].y;
        if (w != 0.f) {
          x[0] += w * y[i][0];
          x[1] += w * y[i][1];
        }
      }
    }
    float* to = tile[way] + (lane & 31) * LD + 16 * (wave_id() % NB) + 4 * (lane >> 5);
    store4(to, x[0]);
    store4(to + 8, x[1]);
    if (wave_id() % NB == 0 && lane < 32) {
      ms[way][lane] = m;
      ss[way][lane] = sum;
    }
  }
  // and the own tokens', four columns of a row a thread.
  constexpr int RT = COLS / 4;  // threads of a row
  const bool mine = threadIdx.x < 32 * RT;
  const int r = threadIdx.x / RT % 32, c4 = 4 * (threadIdx.x % RT), c = COLS * cb + c4, row = min(r0 + r, rows - 1);
  const int seq = b * f.share + row / each, place = row % each;
  const bool here = r0 + r < rows && c < d.dc;
  f32x4 x = zero4();
  float m = -INFINITY, sum = 0.f;
  {
    const Parts<true> ps(d, kv_lens, seq);
    const float* st = stat + 2 * (((int64_t)seq * d.slots + d.slot0) * each + place);
    const float* own = part + ((int64_t)seq * (d.slots - d.part0) * each + place) * d.dc + min(c, d.dc - 4);
    const int n = mine ? ps.all - ps.front : 0;
    for (int s0 = 0; s0 < n; s0 += 8) {
      f32x4 y[8];
      float2 a[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = min(s0 + i, n - 1);
        a[i] = *reinterpret_cast<const float2*>(st + 2 * (int64_t)s * each);
        y[i] = *reinterpret_cast<const f32x4*>(own + (int64_t)s * each * d.dc);
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) mn = fmaxf(mn, s0 + i < n ? a[i].x : -INFINITY);
      const float ref = mn == -INFINITY ? 0.f : mn, fade = fast_exp2(m - ref);
      m = mn;
      sum *= fade;
      x *= fade;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = s0 + i < n ? fast_exp2(a[i].x - ref) : 0.f;
        sum += w * a[i].y;
        if (w != 0.f) x += w * y[i];
      }
    }
  }
  __syncthreads();
  if (!mine) return;
  float mf = ms[0][r], sf = 0.f;
#pragma unroll
  for (int i = 1; i < WAYS; ++i) mf = fmaxf(mf, ms[i][r]);
  const float rf = mf == -INFINITY ? 0.f : mf, all = fmaxf(m, mf);
  f32x4 front = zero4();
#pragma unroll
  for (int i = 0; i < WAYS; ++i) {
    const float w = fast_exp2(ms[i][r] - rf);
    front += w * *reinterpret_cast<const f32x4*>(tile[i] + r * LD + c4);
    sf += w * ss[i][r];
  }
  if (COLS == 64 && shift) {
    float dot = 0.f;
    if (here) {
      const bf16x4 lo = *reinterpret_cast<const bf16x4*>(qa + (((int64_t)seq * each + place) * 2 + 1) * (d.dc + d.dr) + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) dot += (float)lo[j] * front[j];
    }
#pragma unroll
    for (int i = 1; i < RT; i *= 2) dot += __shfl_xor(dot, i);
    float* to = shift + ((int64_t)seq * each + place) * 8;
    if (r0 + r < rows && c4 == 0) {
      to[cb] = sf == 0.f ? 0.f : dot / sf * d.scale * kLog2e;
      if constexpr (CB < 8) to[CB + cb] = 0.f;
    }
  }
  if (!here) return;
  const float ref = all == -INFINITY ? 0.f : all, wf = fast_exp2(mf - ref), wo = fast_exp2(m - ref);
  const float total = wf * sf + wo * sum;
  store4(olat + ((int64_t)seq * each + place) * d.dc + c, (wf * front + wo * x) * (total == 0.f ? 0.f : 1.f / total));
}

static int prefix_blocks(const DecDims& d) { return (int)(((int64_t)d.share * d.n * d.H + kPreRows - 1) / kPreRows); }
// Rows of 32 times splits: each leaves 64 or 32 KB.
static size_t prefix_tiles(const DecDims& d, int units) { return (size_t)units * prefix_blocks(d) * 4 * d.splits; }
static size_t tile_bytes(const DecDims& d) { return 32 * (d.dc > 256 ? 512 : 256) * sizeof(float); }

// Rows from 33 on (40 rows over 4096 tokens, us with the join: 21, latent_split and its join 30; 32 rows: 20 and 22),
// prefixes whose table has 4096 tokens or more (the host does not know their lengths), 32-bit row numbers in LDS.
//
// The tokens are divided by what was measured, in us: a workgroup takes 10.5 and 0.061 a token, one over own tokens 7.5
// and 0.065, the join 0.11 a split (measured with parts of half the bytes; with 0.2 four of ten shapes were 1 to 2 us
// shorter and four as much longer).  With fewer than 256 the own tokens fill the other CUs.  `least` is what a perfect
// division of all of it would take; `longest` what it takes if every own workgroup is as long as its share of the table:
// CUs without a prefix run own ones meanwhile, what is left follows in rounds.  (64 sequences of 16 heads, 8192 and up to
// 1024 tokens, launch and join: 59 in splits of 256, 51 of 512, 74 of 1024, 63 of 384; 32768 and 512: 102 of 1024, 108 of
// 1184, 112 of 1280, 133 of 896; 4 prefixes of 4096, 512 rows each: 55 of 256, 49 of 384, 50 of 512.)
bool prefix_plan(DecDims& d, int units, const DecDims& own) {
  const int64_t rows = (int64_t)d.share * d.n * d.H, most = (int64_t)d.table * d.page;
  if (rows <= 32 || most < kPreTable || (int64_t)d.pages * d.page > UINT32_MAX) return false;
  const int64_t blocks = (int64_t)prefix_blocks(d) * units;
  const int64_t others = (int64_t)own.splits * own.groups * own.B;
  const double other = 0.065 * own.chunk + 7.5;
  double best = 0;
  for (int chunk = 64; chunk <= kPreChunk; chunk += 32) {
    const int64_t splits = (most + chunk - 1) / chunk, wg = blocks * splits;
    const double each = 0.061 * chunk + 10.5, rounds = (double)((wg + 255) / 256) * each;
    const double all = ((double)wg * each + (double)others * other) / 256, least = rounds > all ? rounds : all;
    const int64_t meanwhile = wg % 256 ? (256 - wg % 256) * (int64_t)(each / other + 0.15) : 0;
    const double longest = rounds + (double)(((others > meanwhile ? others - meanwhile : 0) + 255) / 256) * other;
    const double cost = 0.7 * least + 0.3 * longest + 0.11 * (double)splits;
    if (chunk == 64 || cost < best) {
      best = cost;
      d.chunk = chunk;
    }
  }
  d.splits = (int)((most + d.chunk - 1) / d.chunk);
  return blocks * d.splits <= (1 << 30);
}

size_t prefix_bytes(const DecDims& d, int units) { return prefix_tiles(d, units) * tile_bytes(d); }

void launch_prefix(const PrefixCall& c, bool scored, hipStream_t st) {
  const int blocks = prefix_blocks(c.f);
  const int own = c.d.splits * c.d.groups * c.d.B, front = c.f.splits * c.units * blocks;
  const int early = front < 256 ? 0 : (own / 2 < 128 ? own / 2 : 128) & ~7;  // (whole rounds of the XCDs)
  const unsigned grid = (unsigned)(own + front);
  auto go = [&](auto m, auto s) {
    constexpr int MT = decltype(m)::value;
    constexpr bool SCORED = decltype(s)::value != 0;
    if (c.f.dc > 256)
      hipLaunchKernelGGL((latent_prefix<512, MT, SCORED>), dim3(grid), dim3(256), 0, st, c, blocks, early,
                         (f32x4*)c.parts);
    else
      hipLaunchKernelGGL((latent_prefix<256, MT, SCORED>), dim3(grid), dim3(256), 0, st, c, blocks, early,
                         (f32x4*)c.parts);
  };
  auto rows = [&](auto s) {
    if (c.own_tiles == 1) go(IntC<1>(), s);
    else if (c.own_tiles == 2) go(IntC<2>(), s);
    else go(IntC<4>(), s);
  };
  if (scored) rows(IntC<1>());
  else rows(IntC<0>());
}

void launch_prefix_join(const PrefixCall& c, hipStream_t st, float* shift) {
  const int blocks = prefix_blocks(c.f);
  auto run = [&](auto dc, auto cols, auto ways) {
    constexpr int DC = decltype(dc)::value, COLS = decltype(cols)::value, WAYS = decltype(ways)::value;
    hipLaunchKernelGGL((latent_prefix_join<DC, COLS, WAYS>), dim3((unsigned)(c.units * blocks * 4 * (DC / COLS))),
                       dim3(4 * COLS * WAYS), 0, st, c.f, c.d, blocks, (const f32x4*)c.parts, c.part, c.stat, c.lens,
                       c.olat, c.qa, shift);
  };
  // Where 64 columns a workgroup leave half of the CUs without one, 16: a CU takes in about 10 bytes a clock.  (Us, 64
  // rows of 512 latents in 64 splits: 11.3 and 5.9; 512 rows, 128 workgroups: 14.5 and 12.1; 1024 rows in 32 splits, 256
  // workgroups: 15.0 and 16.5.)
  const int64_t rows = (int64_t)c.f.share * c.f.n * c.f.H;
  const bool few = c.units * ((rows + 31) / 32) * ((c.f.dc + 63) / 64) <= 128 && !shift;
  auto go = [&](auto dc) {
    if (few) run(dc, IntC<16>(), IntC<8>());
    else run(dc, IntC<64>(), IntC<2>());
  };
  if (c.f.dc > 256) go(IntC<512>());
  else go(IntC<256>());
}

}  // namespace ah
