// What the kernels of the absorbed form share: the sizes of a call and how the tokens of
// its sequences and prefixes are divided.
#pragma once
#include "latent.hpp"

namespace ah {

// Keep a value in the accumulator half of the register file.
template <typename F> __device__ __forceinline__ void in_accum(F& x) { asm volatile("" : "+a"(x)); }

struct DecDims {
  int B, n, H, dn, dr, dv, dc, page, pages, table, rope, inter;
  int chunk, splits, groups;  // tokens a split (whole tiles), splits of the longest sequence, row groups
  float scale;
  int64_t qs[3];
  int share;         // latent_split: sequences whose rows read the same tokens (those of a prefix, or one)
  int slot0, slots;  // its first slot among a row's parts, and all of them
  int qn;            // rows that a query takes in q_lat: it, and where asked for what its rounding left out
  int part0;         // slots before the first whose part lies row by row (latent_prefix leaves its parts in its own order)
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
// The parts of sequence b's rows: those of the prefix's splits, then those of its own.  (Whether there are
// prefixes is known when a kernel is compiled: with the question asked in it, latent_up's join of 16 rows was
// 1 us longer in the calls that have none.)
template <bool FRONT>
struct Parts {
  int front, all, skip;  // splits of the prefix, of both, slots to leave out between them
  __device__ __forceinline__ Parts(const DecDims& d, const int32_t* kv_lens, int b) {
    front = FRONT ? (pre_len(d, b) + d.pre_chunk - 1) / d.pre_chunk : 0;
    all = front + (!FRONT || d.splits ? (dec_len(d, kv_lens, b) + d.chunk - 1) / d.chunk : 0);
    skip = FRONT ? d.pre_splits - front : 0;
  }
  __device__ __forceinline__ int slot(int s) const { return s < front ? s : s + skip; }
};

// Eight zeros: the source of the padding of a latent narrower than its tile.
static __device__ __attribute__((aligned(16))) const uint32_t lat_zeros[8] = {0, 0, 0, 0, 0, 0, 0, 0};

// 16 x 16 fragments of eight k values a lane (row operand) and of the four
// tokens 4 g + j that a result's registers hold (column operand).
template <typename T> struct M16;
template <> struct M16<bf16> {
  typedef bf16x8 frag;
  typedef bf16x4 half;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma4(half a, half b, f32x4 c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
  }
};
template <> struct M16<float> {
  typedef f32x8 frag;
  typedef f32x4 half;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ f32x4 mma4(half a, half b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};
template <typename T, int W>
struct DTile : LTile<T, W, 16> {
  typedef LTile<T, W, 16> L;
  // (from base addresses as in LTile: row16_base and col16_base plus the tile's LDS address)
  static __device__ __forceinline__ uint32_t row16_base() {
    return L::off(lane_id() & 15, 8 / L::VEC * (lane_id() >> 4));
  }
  static __device__ __forceinline__ typename M16<T>::frag row16(uint32_t base, int k0) {
    typedef const __attribute__((address_space(3))) char* lds_p;
    const int c = k0 / L::VEC;
    if constexpr (sizeof(T) == 2) {
      return *(const __attribute__((address_space(3))) bf16x8*)((lds_p)(base ^ L::piece(c)) + L::above(c));
    } else {
      const f32x4 a = *(const __attribute__((address_space(3))) f32x4*)((lds_p)(base ^ L::piece(c)) + L::above(c));
      const f32x4 b = *(const __attribute__((address_space(3))) f32x4*)((lds_p)(base ^ L::piece(c + 1)) + L::above(c));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  static __device__ __forceinline__ uint32_t col16_base() {
    const int l = lane_id(), t = l & 15, g = l >> 4;
    if constexpr (sizeof(T) == 2) return L::off(4 * g + (t >> 2), (t & 3) >> 1) + 8 * (t & 1);
    else return L::off(4 * g, t >> 2) + 4 * (t & 3);
  }
  static __device__ __forceinline__ typename M16<T>::half col16(uint32_t base, int c0) {
    typedef const __attribute__((address_space(3))) char* lds_p;
    const int c = c0 / L::VEC;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) bf16x4* v4_p;
      return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((v4_p)((lds_p)(base ^ L::piece(c)) + L::above(c)));
    } else {
      f32x4 z;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const lds_p p = (lds_p)(base ^ L::piece(c) ^ (L::swz(j) << 4)) + j * L::ROWB + L::above(c);
        z[j] = *(const __attribute__((address_space(3))) float*)p;
      }
      return z;
    }
  }
};

// One split of one sequence against 16 MT of its query rows (row t H + h).  NW
// waves go over tiles of 16 NW tokens: wave w loads 16 tokens of each tile and
// computes with the 16 rows w % MT and the tokens of MT waves.  The waves of a
// row group join at the end.
//
// Bound by the cache's bytes: 16 heads need 44 operations a byte (30, and 14 for the
// probabilities' second number).  So the tiles go straight to LDS, two of them (with 512
// bf16 latents 74 KB at two waves, so two workgroups a CU, and 147 KB at four), and a
// wave that has its rows to itself (MT = 1) never meets a barrier: it loads what it
// reads.  The split's page numbers lie in LDS, so no wait for an index drains the tiles
// in flight.  64 sequences of up to 8192 tokens, 16 heads: 95 to 97 us for 440 MB,
// 4.6 TB/s; 4 of 32768: 33 us, 4.6 TB/s; both where a copy reaches 5.0.
//
// (With 512 latents the accumulators take 128 registers and the query's fragments 144 in
// float32 and 144 in bf16 where it enters as two numbers.  The accumulators are held where they are while
// they fade: else the compiler copies all of them ahead of that, and puts up to 97 registers into
// scratch memory, which it did not always get back whole.)
//
// The rows of a launch are those of `share` sequences after one another: one, or all that
// follow the same prefix (`own`, then, are the lengths of what follows it).  With SCORED the
// query enters as two bf16 numbers, and where `score` is given the scores in powers of
// two are left there for latent_weigh, a wave's 16 x 16 of them as they lie in its registers.
template <typename T, int DC, int NW> struct SplitLds {
  static constexpr int SC = 16 * DTile<T, DC>::ROWB, SR = 16 * DTile<T, 64>::ROWB;  // one wave's tokens of a tile
  // two tiles, or one where they do not fit (float32 with four waves, bound by its matrix instructions: 624 rows over
  // 2952 tokens 63 us, with two waves and two tiles 151)
  static constexpr int NB = sizeof(T) * NW <= 8 ? 2 : 1;
  char sk[NB * NW * (SC + SR)];
  int32_t spt[kDecPages];
  float sm[NW][16], ss[NW][16];
};
// Split `sp` of unit b (a sequence, or with FRONT a prefix too) against row group `rg` of its rows.
template <typename T, int DC, int MT, int NW, bool SCORED, bool FRONT>
__device__ __forceinline__ void split_tokens(const DecDims& d, SplitLds<T, DC, NW>& lds, int sp, int rg, int b,
                                             const T* __restrict__ qa,
                                             const T* __restrict__ cache, const int32_t* __restrict__ table,
                                             const int32_t* __restrict__ kv_lens, const int32_t* __restrict__ own,
                                             int own_most, float* __restrict__ part, float* __restrict__ stat,
                                             float* __restrict__ olat, float* __restrict__ score) {
  constexpr int DR = 64, W = DC + DR, KS = W / 32, NT = DC / 16, TK = 16 * NW, TW = NW / MT, V = 16 / (int)sizeof(T);
  constexpr int NP = sizeof(T) == 2 ? 2 : 1;    // operands of a probability
  constexpr int NQ = SCORED && sizeof(T) == 2 ? 2 : 1;  // and of a query
  constexpr int PC = DC / V, PR = DR / V;       // pieces of a row's latent and rotated key
  constexpr int IC = PC * 16 / 64, IR = PR * 16 / 64;  // loads of one wave for its 16 tokens
  typedef DTile<T, DC> LC;
  typedef DTile<T, DR> LR;
  typedef typename M16<T>::frag frag;
  typedef typename M16<T>::half half;
  constexpr int SC = SplitLds<T, DC, NW>::SC, SR = SplitLds<T, DC, NW>::SR, NB = SplitLds<T, DC, NW>::NB;
  char* const sk = lds.sk;
  int32_t* const spt = lds.spt;
  float(*const sm)[16] = lds.sm;
  float(*const ss)[16] = lds.ss;
  const int wv = wave_id(), lane = lane_id(), rw = wv % MT, tw = wv / MT;
  const int len = dec_len(d, kv_lens, b), each = d.n * d.H, rows = (FRONT ? d.share : 1) * each, wide = d.dc + d.dr;
  const int first = sp * d.chunk, end = min(len, first + d.chunk);
  if (first >= len && (sp > 0 || d.slots > 1)) return;  // (one split only: it writes the empty sequence's zeros)
  const int page0 = first / d.page;
  for (int i = threadIdx.x; first < end && i <= (end - 1) / d.page - page0; i += 64 * NW)
    spt[i] = min(max(table[(int64_t)b * d.table + page0 + i], 0), d.pages - 1);
  const int row = 16 * (rg * MT + rw) + (lane & 15);
  int seq = b, place = min(row, rows - 1);  // this lane's row: its sequence, and its place there
  if (FRONT && d.share > 1) {
    seq = b * d.share + place / each;
    place %= each;
  }
  int seen = len - d.n + place / d.H + 1;  // tokens that it sees
  if (FRONT && own) seen += min(max(own[seq], 0), own_most);
  const int least = len - d.n + 1;  // and that every row sees
  const T* qr = qa + ((int64_t)seq * each + place) * d.qn * wide;
  frag qf[NQ][KS];
#pragma unroll
  for (int u = 0; u < NQ; ++u)
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const int k = 32 * t + 8 * (lane >> 4);
      if (32 * t < DC) qf[u][t] = ld_frag(k < d.dc ? qr + u * wide + k : (const T*)lat_zeros);
      else qf[u][t] = ld_frag(k - DC < d.dr ? qr + u * wide + d.dc + k - DC : (const T*)lat_zeros);
    }
  __syncthreads();  // the page numbers are there
  const uint32_t lds0 = lds_addr(sk);
  constexpr int RL = PC >= 64 ? PC / 64 : 1;  // loads a row
  // Byte offset of this lane's piece in load l of a row with swizzle z.  The padding
  // of a width reads the row's first piece instead: the query has zeros there.
  auto piece = [&](int l, int z) {
    const int c = 64 * l + (lane ^ z);
    return c * V < d.dc ? 16 * c : 0;
  };
  uint32_t oc[16];
  if constexpr (RL == 1) {
#pragma unroll
    for (int z = 0; z < 16; ++z) oc[z] = piece(0, z);
  }
  // this wave's 16 tokens of the tile at k0 into buffer `buf`; tokens past the end repeat the last one (masked below)
  auto load = [&](int k0, int buf) {
    const int j = min(k0 + 16 * wv + (lane & 15), end - 1), pg = j / d.page;
    const uint64_t at = (uint64_t)(cache + ((int64_t)spt[pg - page0] * d.page + (j - pg * d.page)) * wide);
    const uint32_t lo = (uint32_t)at, hi = (uint32_t)(at >> 32);
    const uint32_t dst = lds0 + (buf * NW + wv) * (SC + SR);
#pragma unroll
    for (int i = 0; i < IC; ++i) {  // 64 pieces of the 16 rows of PC
      if constexpr (PC >= 64) {
        const int r = i / RL;
        const uint64_t row = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, r) << 32 |
                             (uint32_t)__builtin_amdgcn_readlane(lo, r);
        dma16_raw_s(row, RL == 1 ? oc[r] : piece(i % RL, r), dst + 1024 * i);  // (swz(r) = r)
      } else {
        const int r = (64 * i + lane) / PC;
        const uint64_t row = (uint64_t)__shfl(hi, r) << 32 | (uint32_t)__shfl(lo, r);
        const int c = (lane % PC) ^ LC::swz(r);
        dma16_raw((const void*)(row + (c * V < d.dc ? 16 * c : 0)), dst + 1024 * i);
      }
    }
#pragma unroll
    for (int i = 0; i < IR; ++i) {
      const int e = 64 * i + lane, r = e / PR, c = (e % PR) ^ LR::swz(r);
      const uint64_t row = (uint64_t)__shfl(hi, r) << 32 | (uint32_t)__shfl(lo, r);
      dma16_raw((const void*)(row + d.dc * sizeof(T) + (c * V < d.dr ? 16 * c : 0)), dst + SC + 1024 * i);
    }
  };
  f32x4 acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = zero4();
  const float c2 = d.scale * kLog2e;
  float m = -INFINITY, sum = 0.f;
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // the query fragments: no later wait for them drains the tiles
  if (first < end) load(first, 0);
  if (NB == 2 && first + TK < end) load(first + TK, 1);
  int buf = 0;
  for (int k0 = first; k0 < end; k0 += TK, buf ^= NB - 1) {
    if (NB == 2 && k0 + TK < end) vm_wait<IC + IR>();  // this tile is there, the next one in flight
    else vm_wait<0>();
    if constexpr (MT > 1) bare_barrier();
    f32x4 s[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint32_t kc = lds0 + (buf * NW + MT * tw + i) * (SC + SR);
      uint32_t rc = kc + LC::row16_base(), rr = kc + SC + LR::row16_base();
      asm volatile("" : "+v"(rc), "+v"(rr));
      f32x4 x[2] = {zero4(), zero4()};  // two chains: each waits for its own result only
      in_groups<KS, sizeof(T) == 2 ? 6 : 2, frag>(
          [&](int t) { return 32 * t < DC ? LC::row16(rc, 32 * t) : LR::row16(rr, 32 * t - DC); },
          [&](int t, frag a) {
#pragma unroll
            for (int u = 0; u < NQ; ++u) x[(t ^ u) & 1] = M16<T>::mma(a, qf[u][t], x[(t ^ u) & 1]);
          });
      s[i] = x[0] + x[1];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) s[i] *= c2;
    if (k0 + TK > min(end, least)) {
      const int lim = min(end, seen) - k0 - 16 * MT * tw;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (16 * i + tile_row(r) >= lim) s[i][r] = -INFINITY;
    }
    if constexpr (SCORED) {
      if (score) {  // (tiles past the end have no place)
        const int tiles = (d.table * d.page + 15) / 16;
        const int64_t at = (int64_t)b * (d.groups * MT) + rg * MT + rw;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int tile = k0 / 16 + MT * tw + i;
          if (16 * tile < end) store4(score + ((at * tiles + tile) * 64 + lane) * 4, s[i]);
        }
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[i][r]);
    if (__any(top > m + kLag)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float mn = fmaxf(m, top), fade = mn == -INFINITY ? 1.f : fast_exp2(m - mn);
      m = mn;
      sum *= fade;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        in_accum(acc[n]);
        acc[n] *= fade;
        in_accum(acc[n]);
      }
    }
    const float ref = m == -INFINITY ? 0.f : m;  // a row that has seen nothing yet: every p is exp2(-inf) = 0
    half p[NP][MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float e = fast_exp2(s[i][r] - ref);
        sum += e;
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          p[k][i][r] = (T)e;
          e -= (float)p[k][i][r];
        }
      }
    uint32_t cc = lds0 + buf * NW * (SC + SR) + MT * tw * (SC + SR) + LC::col16_base();
    asm volatile("" : "+v"(cc));
    if constexpr (MT == 1) {
      in_groups<NT, sizeof(T) == 2 ? 8 : 2, half>([&](int n) { return LC::col16(cc, 16 * n); },
                                               [&](int n, half a) {
#pragma unroll
                                                 for (int k = 0; k < NP; ++k) acc[n] = M16<T>::mma4(a, p[k][0], acc[n]);
                                               });
    } else {  // 32 tokens an instruction
#pragma unroll
      for (int i = 0; i < MT; i += 2) {
        frag pp[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) pp[k] = __builtin_shufflevector(p[k][i], p[k][i + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        const uint32_t ca = cc + i * (SC + SR);
        in_groups<NT, sizeof(T) == 2 ? 4 : 1, frag>(
            [&](int n) {
              return __builtin_shufflevector(LC::col16(ca, 16 * n), LC::col16(ca + SC + SR, 16 * n), 0, 1, 2, 3,
                                             4, 5, 6, 7);
            },
            [&](int n, frag a) {
#pragma unroll
              for (int k = 0; k < NP; ++k) acc[n] = M16<T>::mma(a, pp[k], acc[n]);
            });
      }
    }
    // every read of this buffer has returned before it is loaded again
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if constexpr (MT > 1) bare_barrier();
    if (k0 + NB * TK < end) load(k0 + NB * TK, buf);
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  // the TW waves of a row group: a common maximum, then sums pairwise through LDS
  if constexpr (TW > 1) {
    if (lane < 16) {
      sm[wv][lane] = m;
      ss[wv][lane] = sum;
    }
    __syncthreads();
    const int col = lane & 15;
    float mm = -INFINITY;
#pragma unroll
    for (int t = 0; t < TW; ++t) mm = fmaxf(mm, sm[t * MT + rw][col]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    sum = 0.f;
#pragma unroll
    for (int t = 0; t < TW; ++t) sum += ss[t * MT + rw][col] * fast_exp2(sm[t * MT + rw][col] - ref);
    const float fade = fast_exp2(m - ref);
    m = mm;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] *= fade;
    f32x4* x = reinterpret_cast<f32x4*>(sk);
#pragma unroll
    for (int hw = TW / 2; hw; hw >>= 1) {
      __syncthreads();
      if (tw >= hw && tw < 2 * hw) {
#pragma unroll
        for (int n = 0; n < NT; ++n) x[(((tw - hw) * MT + rw) * NT + n) * 64 + lane] = acc[n];
      }
      __syncthreads();
      if (tw < hw) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n] += x[((tw * MT + rw) * NT + n) * 64 + lane];
      }
    }
  }
  if (tw != 0 || row >= rows) return;
  const int64_t at = ((int64_t)seq * d.slots + d.slot0 + sp) * each + place;
  float* dst = part + (((int64_t)seq * (d.slots - d.part0) + d.slot0 - d.part0 + sp) * each + place) * d.dc;
  float by = 1.f;
  if (d.slots == 1) {  // nothing to join
    by = sum == 0.f ? 0.f : 1.f / sum;
    dst = olat + ((int64_t)seq * each + place) * d.dc;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = 16 * n + tile_row(0);
    if (c < d.dc) store4(dst + c, acc[n] * by);
  }
  if (lane < 16 && (SCORED || d.slots > 1)) {
    stat[2 * at] = m;
    stat[2 * at + 1] = sum;
  }
}

// latent_prefix: the prefixes' tokens against the rows of all sequences that follow them,
// and each sequence's own tokens, in one launch (bf16).
struct PrefixCall {
  DecDims f, d;  // over the prefixes, and the own tokens
  int units;     // prefixes
  int own_tiles;  // row tiles of a workgroup of split_tokens over the own tokens
  const bf16 *qa, *cache;
  const int32_t *prefix_table, *prefix_lens, *table, *lens;
  float *part, *stat, *olat, *score;
  void* parts;   // of the prefixes, prefix_bytes
};
// Whether it takes the rows of `units` prefixes, beside the own tokens `own`; divides their tokens for it, if so.
bool prefix_plan(DecDims& d, int units, const DecDims& own);
// Bytes of the parts that it leaves for the join.
size_t prefix_bytes(const DecDims& d, int units);
void launch_prefix(const PrefixCall& c, bool scored, hipStream_t st);
// Joins them with those of the own tokens.  `shift`, unless NULL: a correction of each
// row's sum over the prefix (in its kernel's comment), in eight shares.
void launch_prefix_join(const PrefixCall& c, hipStream_t st, float* shift);

}  // namespace ah
