// Latent attention over a paged cache for gfx950: the append with its rotation,
// and the absorbed form for single tokens (or a few a sequence).
//
//   q_lat[h] = w_kv[h, :dn]^T q_nope[h]                      (absorb)
//   s_j = scale (q_lat . c_j + rotate(q_pe) . k_j)           (split over the tokens)
//   o_lat = sum_j softmax(s)_j c_j                           (joined in the last kernel)
//   o[h] = w_kv[h, dn:] o_lat[h]                             (up)
//
// All heads of a sequence read the same cache row, once, as key and as value.
// q_lat is rounded to the operand type, as the MFMA takes it; the probabilities
// and o_lat, fp32, enter their products as the sum of two bf16 numbers (the cache's
// bytes leave the matrix instructions idle; with probabilities of eight bits o was off
// by 0.0025 of its norm at 64 sequences of up to 8192 tokens, now by 0.0023, of which
// its own rounding is 0.0017 and q_lat's most of the rest).
#include "latent.hpp"

namespace ah {

// ------------------------------------------------------------------- append
struct AppDims {
  int N, H, dn, dr, dc, page, pages, rope, inter;
  int64_t cs, ks, qs[2];
  unsigned blocks_c;  // workgroups of the cache part, the others rotate q
};

// Four pairs of one row: elements 8 u .. 8 u + 7 (interleaved) or 4 u .. + 3 of both halves.
template <typename T> struct Vec4;
template <> struct Vec4<bf16> { typedef bf16x4 t; };
template <> struct Vec4<float> { typedef f32x4 t; };
template <typename T>
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
    store4(y1 + a, o0);
    store4(y1 + b, o1);
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
struct DecDims {
  int B, n, H, dn, dr, dv, dc, page, pages, table, rope, inter;
  int chunk, splits, groups;  // tokens a split (whole tiles), splits of the longest sequence, row groups
  float scale;
  int64_t qs[3];
};
constexpr int kDecChunk = 1024, kDecPages = kDecChunk + 1;  // tokens of a split, pages that they can lie in
__device__ __forceinline__ int dec_len(const DecDims& d, const int32_t* kv_lens, int b) {
  return (int)min((int64_t)max(kv_lens[b], 0), (int64_t)d.table * d.page);
}

// q_lat [B n, H, dc | rotated q_pe]: a head, 16 query tokens and 64 latent
// columns a workgroup, 16 columns a wave; one more column block rotates.  Latency: 4 to
// 6 us with 4 to 64 sequences of 16 heads (4 MB of weights).
template <typename T>
__global__ __launch_bounds__(256) void latent_absorb(DecDims d, const T* __restrict__ q, const T* __restrict__ w_kv,
                                                     const int32_t* __restrict__ kv_lens,
                                                     const float* __restrict__ cos, const float* __restrict__ sin,
                                                     T* __restrict__ qa) {
  constexpr int V = 16 / (int)sizeof(T), LW = 64 + V, LQ = 128 + V;
  __shared__ __attribute__((aligned(16))) T sw[128 * LW];
  __shared__ __attribute__((aligned(16))) T sq[16 * LQ];
  const int h = blockIdx.x, c0 = 64 * blockIdx.y, r0 = 16 * blockIdx.z, R = d.B * d.n, wide = d.dc + d.dr;
  if (c0 >= d.dc) {
    for (int e = threadIdx.x; e < 16 * (d.dr / 8); e += 256) {
      const int r = r0 + e / (d.dr / 8), u = e % (d.dr / 8);
      if (r >= R) break;
      const T* x = q + r / d.n * d.qs[0] + r % d.n * d.qs[1] + h * d.qs[2] + d.dn;
      T* y = qa + ((int64_t)r * d.H + h) * wide + d.dc;
      if (cos) {
        const int64_t p = min(max(dec_len(d, kv_lens, r / d.n) - d.n + r % d.n, 0), d.rope - 1);
        rotate4(x, cos + p * (d.dr / 2), sin + p * (d.dr / 2), u, d.dr, d.inter, y, (T*)nullptr);
      } else {
        float t[8];
        load8(x + 8 * u, t);
        store8(y + 8 * u, t);
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
  if (r < R && c < d.dc) store4(qa + ((int64_t)r * d.H + h) * wide + c, z);
}

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

// Eight zeros: the source of the padding of a latent narrower than its tile.
__device__ __attribute__((aligned(16))) const uint32_t lat_zeros[8] = {0, 0, 0, 0, 0, 0, 0, 0};

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
// (float32 with 512 latents: the query's fragments take 144 registers and the
// accumulators 128; 3 registers lie in scratch memory with MT = 1, 54 with MT = 2.)
template <typename T, int DC, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void latent_split(DecDims d, const T* __restrict__ qa,
                                                        const T* __restrict__ cache, const int32_t* __restrict__ table,
                                                        const int32_t* __restrict__ kv_lens, float* __restrict__ part,
                                                        float* __restrict__ stat, float* __restrict__ olat) {
  constexpr int DR = 64, W = DC + DR, KS = W / 32, NT = DC / 16, TK = 16 * NW, TW = NW / MT, V = 16 / (int)sizeof(T);
  constexpr int NP = sizeof(T) == 2 ? 2 : 1;    // operands of a probability
  constexpr int PC = DC / V, PR = DR / V;       // pieces of a row's latent and rotated key
  constexpr int IC = PC * 16 / 64, IR = PR * 16 / 64;  // loads of one wave for its 16 tokens
  typedef DTile<T, DC> LC;
  typedef DTile<T, DR> LR;
  typedef typename M16<T>::frag frag;
  typedef typename M16<T>::half half;
  constexpr int SC = 16 * LC::ROWB, SR = 16 * LR::ROWB;  // one wave's tokens of a tile
  __shared__ __attribute__((aligned(1024))) char sk[2 * NW * (SC + SR)];
  __shared__ int32_t spt[kDecPages];
  __shared__ float sm[NW][16], ss[NW][16];
  const int sp = blockIdx.x, b = blockIdx.z, wv = wave_id(), lane = lane_id(), rw = wv % MT, tw = wv / MT;
  const int len = dec_len(d, kv_lens, b), rows = d.n * d.H, wide = d.dc + d.dr;
  const int first = sp * d.chunk, end = min(len, first + d.chunk);
  if (first >= len && (sp > 0 || d.splits > 1)) return;  // (one split only: it writes the empty sequence's zeros)
  const int page0 = first / d.page;
  for (int i = threadIdx.x; first < end && i <= (end - 1) / d.page - page0; i += 64 * NW)
    spt[i] = min(max(table[(int64_t)b * d.table + page0 + i], 0), d.pages - 1);
  const int row = 16 * (blockIdx.y * MT + rw) + (lane & 15);
  const int seen = len - d.n + min(row, rows - 1) / d.H + 1;  // tokens that this lane's row sees
  const int least = len - d.n + 1;                            // and that every row sees
  const T* qr = qa + ((int64_t)b * rows + min(row, rows - 1)) * wide;
  frag qf[KS];
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    const int k = 32 * t + 8 * (lane >> 4);
    if (32 * t < DC) qf[t] = ld_frag(k < d.dc ? qr + k : (const T*)lat_zeros);
    else qf[t] = ld_frag(k - DC < d.dr ? qr + d.dc + k - DC : (const T*)lat_zeros);
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
  if (first + TK < end) load(first + TK, 1);
  int buf = 0;
  for (int k0 = first; k0 < end; k0 += TK, buf ^= 1) {
    if (k0 + TK < end) vm_wait<IC + IR>();  // this tile is there, the next one in flight
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
          [&](int t, frag a) { x[t & 1] = M16<T>::mma(a, qf[t], x[t & 1]); });
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
      for (int n = 0; n < NT; ++n) acc[n] *= fade;
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
    if (k0 + 2 * TK < end) load(k0 + 2 * TK, buf);
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
  float* dst = part + (((int64_t)b * d.splits + sp) * rows + row) * d.dc;
  float by = 1.f;
  if (d.splits == 1) {  // nothing to join
    by = sum == 0.f ? 0.f : 1.f / sum;
    dst = olat + ((int64_t)b * rows + row) * d.dc;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = 16 * n + tile_row(0);
    if (c < d.dc) store4(dst + c, acc[n] * by);
  }
  if (lane < 16 && d.splits > 1) {
    const int64_t at = ((int64_t)b * d.splits + sp) * rows + row;
    stat[2 * at] = m;
    stat[2 * at + 1] = sum;
  }
}

// o_lat [B n H, dc]: the splits of a row joined.  16 `ways` threads take 64
// columns of a row, thread group g the splits g, g + ways, ...; the groups join
// through LDS.  (With few rows and many splits the parts are spread over the card
// this way: 4 sequences of 32768 tokens, 16 heads: 16 MB of parts.)
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
    const int ns = (dec_len(d, kv_lens, b) + d.chunk - 1) / d.chunk;
    const int64_t at = (int64_t)b * d.splits * rows + row % rows;
    for (int s = g; s < ns; s += ways) m = fmaxf(m, stat[2 * (at + (int64_t)s * rows)]);
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (int s = g; s < ns; s += ways) {
      const int64_t a = at + (int64_t)s * rows;
      const float w = fast_exp2(stat[2 * a] - ref);
      sum += w * stat[2 * a + 1];
      x += w * *reinterpret_cast<const f32x4*>(part + a * d.dc + c);
    }
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

// o: 16 query tokens of a head times 64 rows of its value projection a
// workgroup, 16 a wave.  With JOIN it joins the splits itself (up to kUpSplits of
// them): where that is a few dozen loads a thread, a launch less is worth more than
// the same parts read once instead of dv / 64 times.  Latency: 5 to 8 us without the join.
constexpr int kUpSplits = 64;
template <typename T, bool JOIN>
__global__ __launch_bounds__(256) void latent_up(DecDims d, const T* __restrict__ w_kv, const float* __restrict__ olat,
                                                 const float* __restrict__ part, const float* __restrict__ stat,
                                                 const int32_t* __restrict__ kv_lens, T* __restrict__ o) {
  constexpr int V = 16 / (int)sizeof(T), LD = 512 + V, PARTS = sizeof(T) == 2 ? 2 : 1, KS = 16;
  __shared__ __attribute__((aligned(16))) T so[PARTS][16 * LD];
  __shared__ float sw[JOIN ? 16 : 1][kUpSplits];
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
    const int ns = (dec_len(d, kv_lens, b) + d.chunk - 1) / d.chunk;
    const float* st = stat + 2 * ((int64_t)b * d.splits * rows + r % d.n * d.H + h);
    float m = -INFINITY, sum = 0.f, ms[kUpSplits / 16], ls[kUpSplits / 16];
#pragma unroll
    for (int i = 0; i < kUpSplits / 16; ++i) {
      const int s = g + 16 * i;
      ms[i] = s < ns ? st[2 * (int64_t)s * rows] : -INFINITY;
      ls[i] = s < ns ? st[2 * (int64_t)s * rows + 1] : 0.f;
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
        const int b = (r0 + r) / d.n, ns = (dec_len(d, kv_lens, b) + d.chunk - 1) / d.chunk;
        const float* p = part + ((int64_t)b * d.splits * rows + (r0 + r) % d.n * d.H + h) * d.dc + c;
#pragma unroll 8
        for (int s = 0; s < ns; ++s) x += sw[r][s] * *reinterpret_cast<const f32x4*>(p + (int64_t)s * rows * d.dc);
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

static int dec_check(const atomic_latent_decode_args* a) {
  if (!a) return ATOMIC_ERR_NULL;
  if (int rc = latent_widths_check(a->dn, a->dr, a->dtype)) return rc;
  if (a->dv < 8 || a->dv > 128 || a->dv % 8 || a->dc < 8 || a->dc > 512 || a->dc % 8 || a->batch < 1 ||
      a->tokens < 1 || a->heads < 1 || (int64_t)a->tokens * a->heads > 4096 || a->page < 1 || a->pages < 1 ||
      a->table_pages < 1 || (a->interleaved != 0 && a->interleaved != 1))
    return ATOMIC_ERR_SHAPE;
  // grid dimensions and token numbers
  if (a->batch > 65535 || (int64_t)a->batch * a->tokens > 65535 * 16 ||
      (int64_t)a->table_pages * a->page > (1 << 30))
    return ATOMIC_ERR_SHAPE;
  if (!whole_pieces({a->q_stride[0], a->q_stride[1], a->q_stride[2]}, a->dtype)) return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}

// Rows a workgroup of latent_split takes, in tiles of 16.
static int dec_row_tiles(const atomic_latent_decode_args* a) {
  const int rows = a->tokens * a->heads;
  return rows <= 16 ? 1 : rows <= 32 || a->dtype != ATOMIC_BF16 ? 2 : 4;
}

static DecDims dec_dims(const atomic_latent_decode_args* a) {
  DecDims d{a->batch, a->tokens, a->heads, a->dn, a->dr, a->dv, a->dc, a->page, a->pages, a->table_pages,
            a->rope_rows, a->interleaved, 0, 0, 0, a->scale, {a->q_stride[0], a->q_stride[1], a->q_stride[2]}};
  const int mt = dec_row_tiles(a), rt = 16 * mt, tile = mt == 4 ? 64 : 32;
  d.groups = (d.n * d.H + rt - 1) / rt;
  // As many workgroups as the card holds at once if every sequence were as long as
  // its table (the host does not know the lengths, so a table wider than the sequences
  // costs parallelism: 64 of 1024 tokens, 16 heads, whole calls: 42 us with a table as
  // wide, 89 with one of 8192 tokens, 293 with one of 131072): two a CU with two waves each in bf16, else one (the tiles' LDS).
  // Split and join together, us: 64 sequences of up to 8192 tokens, 16 heads: 116 in
  // splits of 512, 103 of 1024; 4 of 32768: 42 of 256 or 512, 56 of 128; 8 of 4096
  // with 64 rows: 33 of 128, 36 of 256, 46 of 64; one of 777: 18 of 32, 22 of 128.
  const int64_t slots = mt == 4 || a->dtype != ATOMIC_BF16 ? 256 : 512;
  const int64_t most = (int64_t)d.table * d.page, want = (most * d.B * d.groups + slots - 1) / slots;
  const int64_t chunk = want < tile ? tile : want > kDecChunk ? kDecChunk : want;
  d.chunk = (int)((chunk + tile - 1) / tile * tile);
  d.splits = (int)((most + d.chunk - 1) / d.chunk);
  return d;
}
// Whether latent_up joins the splits: at most 48 loads a thread, in steps of eight
// (25 loads: 14.6 us against 7.4 + 7.2 of two launches, 64: 25.7 against 9 + 10).
static bool dec_up_joins(const DecDims& d) {
  const int64_t rows = (int64_t)d.B * d.n < 16 ? (int64_t)d.B * d.n : 16;
  return d.splits > 1 && d.splits <= kUpSplits && d.splits * ((rows * d.dc / 4 + 255) / 256) <= 48;
}
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }
static size_t dec_qa_bytes(const DecDims& d, int dtype) {
  return up256((size_t)d.B * d.n * d.H * (d.dc + d.dr) * (dtype == ATOMIC_BF16 ? 2 : 4));
}
static size_t dec_olat_bytes(const DecDims& d) { return up256((size_t)d.B * d.n * d.H * d.dc * sizeof(float)); }
// one split needs no parts
static size_t dec_part_rows(const DecDims& d) { return d.splits > 1 ? (size_t)d.B * d.splits * d.n * d.H : 0; }
static size_t dec_stat_bytes(const DecDims& d) { return up256(dec_part_rows(d) * 2 * sizeof(float)); }
static size_t dec_part_bytes(const DecDims& d) { return dec_part_rows(d) * d.dc * sizeof(float); }

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

extern "C" size_t atomic_latent_decode_workspace_size(const atomic_latent_decode_args* a) {
  if (dec_check(a) != ATOMIC_OK) return 0;
  const DecDims d = dec_dims(a);
  return dec_qa_bytes(d, a->dtype) + dec_olat_bytes(d) + dec_stat_bytes(d) + dec_part_bytes(d);
}

template <typename T, int DC>
static void launch_split(const DecDims& d, int mt, hipStream_t st, const T* qa, const void* cache, const int32_t* table,
                         const int32_t* kv_lens, float* part, float* stat, float* olat) {
  const dim3 grid((unsigned)d.splits, (unsigned)d.groups, (unsigned)d.B);
  auto go = [&](auto m) {
    constexpr int NW = decltype(m)::value == 4 ? 4 : 2;
    hipLaunchKernelGGL((latent_split<T, DC, decltype(m)::value, NW>), grid, dim3(64 * NW), 0, st, d, qa,
                       (const T*)cache, table, kv_lens, part, stat, olat);
  };
  if (mt == 1) go(IntC<1>());
  else if (mt == 2) go(IntC<2>());
  else if constexpr (sizeof(T) == 2) go(IntC<4>());
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
  const DecDims d = dec_dims(a);
  const hipStream_t st = (hipStream_t)stream;
  Launch L{a->profile, st};
  auto go = [&](auto t) {
    typedef decltype(t) T;
    T* qa = (T*)workspace;
    float* olat = (float*)((char*)workspace + dec_qa_bytes(d, a->dtype));
    float* stat = (float*)((char*)olat + dec_olat_bytes(d));
    float* part = (float*)((char*)stat + dec_stat_bytes(d));
    const unsigned rt = (unsigned)((d.B * d.n + 15) / 16);
    int rc = L("latent_absorb", [&] {
      hipLaunchKernelGGL((latent_absorb<T>), dim3((unsigned)d.H, (unsigned)((d.dc + 63) / 64 + 1), rt), dim3(256), 0,
                         st, d, (const T*)q, (const T*)w_kv, kv_lens, cos, sin, qa);
    });
    if (rc) return rc;
    rc = L("latent_split", [&] {
      if (d.dc <= 256)
        launch_split<T, 256>(d, dec_row_tiles(a), st, qa, cache, page_table, kv_lens, part, stat, olat);
      else
        launch_split<T, 512>(d, dec_row_tiles(a), st, qa, cache, page_table, kv_lens, part, stat, olat);
    });
    if (rc) return rc;
    const bool joins = dec_up_joins(d);
    if (d.splits > 1 && !joins) {
      int ways = 1;  // about four splits a thread
      while (ways < 16 && 4 * ways < d.splits) ways *= 2;
      const int64_t units = (int64_t)d.B * d.n * d.H * ((d.dc + 63) / 64);
      rc = L("latent_join", [&] {
        hipLaunchKernelGGL(latent_join, dim3((unsigned)((units * ways + 15) / 16)), dim3(256), 0, st, d, ways, part,
                           stat, kv_lens, olat);
      });
      if (rc) return rc;
    }
    return L("latent_up", [&] {
      auto go = [&](auto j) {
        hipLaunchKernelGGL((latent_up<T, decltype(j)::value != 0>),
                           dim3((unsigned)d.H, (unsigned)((d.dv + 63) / 64), rt), dim3(256), 0, st, d,
                           (const T*)w_kv, olat, part, stat, kv_lens, (T*)o);
      };
      if (joins) go(IntC<1>());
      else go(IntC<0>());
    });
  };
  return a->dtype == ATOMIC_BF16 ? go(bf16()) : go(float());
}
