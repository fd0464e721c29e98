// Latent attention over a paged cache for gfx950: the append with its rotation,
// and the absorbed form for single tokens (or a few a sequence).
//
//   q_lat[h] = w_kv[h, :dn]^T q_nope[h]                      (absorb)
//   s_j = scale (q_lat . c_j + rotate(q_pe) . k_j)           (split over the tokens)
//   o_lat = sum_j softmax(s)_j c_j                           (joined in the last kernel)
//   o[h] = w_kv[h, dn:] o_lat[h]                             (up)
//
// All heads of a sequence read the same cache row, once, as key and as value.
// q_lat and the probabilities are rounded to the operand type, as the MFMA
// takes them; o_lat stays fp32 to the end (in bf16 it enters the last product as
// the sum of two bf16 numbers).
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

// One 16-byte piece to copy or four pairs to rotate a thread.
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
__device__ __forceinline__ int dec_len(const DecDims& d, const int32_t* kv_lens, int b) {
  return (int)min((int64_t)max(kv_lens[b], 0), (int64_t)d.table * d.page);
}

// q_lat [B n, H, dc | rotated q_pe]: a head, 16 query tokens and 64 latent
// columns a workgroup, 16 columns a wave; one more column block rotates.
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
struct DTile : LTile<T, W> {
  typedef LTile<T, W> L;
  static __device__ __forceinline__ typename M16<T>::frag row16(const char* s, int r0, int k0) {
    const int l = lane_id(), r = r0 + (l & 15), k = k0 + 8 * (l >> 4);
    if constexpr (sizeof(T) == 2) {
      return *reinterpret_cast<const bf16x8*>(s + L::off(r, k / 8));
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(s + L::off(r, k / 4));
      const f32x4 b = *reinterpret_cast<const f32x4*>(s + L::off(r, k / 4 + 1));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  static __device__ __forceinline__ typename M16<T>::half col16(const char* s, int r0, int c0) {
    const int l = lane_id(), t = l & 15, g = l >> 4;
    if constexpr (sizeof(T) == 2) {
      const int r = r0 + 4 * g + (t >> 2), c = c0 + 4 * (t & 3);
      typedef __attribute__((address_space(3))) bf16x4* lds_p;
      return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_p)(s + L::off(r, c / 8) + 2 * (c & 7)));
    } else {
      const int c = c0 + t;
      f32x4 z;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        z[j] = *reinterpret_cast<const float*>(s + L::off(r0 + 4 * g + j, c / 4) + 4 * (c & 3));
      return z;
    }
  }
};

// One split of one sequence against 16 MT of its query rows (row t H + h): tiles
// of 64 tokens, wave w taking the 16 rows w % MT and MT of the tile's four groups
// of 16 tokens.  The waves of a row group join at the end.
template <typename T, int DC, int MT>
__global__ __launch_bounds__(256) void latent_split(DecDims d, const T* __restrict__ qa, const T* __restrict__ cache,
                                                    const int32_t* __restrict__ table,
                                                    const int32_t* __restrict__ kv_lens, float* __restrict__ part,
                                                    float* __restrict__ stat) {
  constexpr int DR = 64, W = DC + DR, KS = W / 32, NT = DC / 16, TK = 64, TW = 4 / MT, V = 16 / (int)sizeof(T);
  typedef DTile<T, W> L;
  typedef typename M16<T>::frag frag;
  typedef typename M16<T>::half half;
  __shared__ __attribute__((aligned(1024))) char sk[TK * L::ROWB];
  __shared__ float sm[4][16], ss[4][16];
  const int sp = blockIdx.x, b = blockIdx.z, wv = wave_id(), rw = wv % MT, tw = wv / MT;
  const int len = dec_len(d, kv_lens, b), rows = d.n * d.H, wide = d.dc + d.dr;
  const int first = sp * d.chunk, end = min(len, first + d.chunk);
  if (first >= len) return;
  const int row = 16 * (blockIdx.y * MT + rw) + (lane_id() & 15);
  const int seen = len - d.n + min(row, rows - 1) / d.H + 1;  // tokens that this lane's row sees
  const T* qr = qa + ((int64_t)b * rows + min(row, rows - 1)) * wide;
  frag qf[KS];
#pragma unroll
  for (int t = 0; t < KS; ++t) {
    const int k = 32 * t + 8 * (lane_id() >> 4);
    qf[t] = zero_frag<T>();
    if (32 * t < DC) {
      if (k < d.dc) qf[t] = ld_frag(qr + k);
    } else if (k - DC < d.dr) {
      qf[t] = ld_frag(qr + d.dc + k - DC);
    }
  }
  f32x4 acc[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = zero4();
  const float c2 = d.scale * kLog2e;
  float m = -INFINITY, sum = 0.f;
  for (int k0 = first; k0 < end; k0 += TK) {
    __syncthreads();
    constexpr int PR = W / V;
    for (int e = threadIdx.x; e < TK * PR; e += 256) {
      const int c = e % PR * V, j = min(k0 + e / PR, end - 1);  // rows past the end repeat the last one, masked below
      const int64_t pg = min(max(table[(int64_t)b * d.table + j / d.page], 0), d.pages - 1);
      const T* src = cache + (pg * d.page + j % d.page) * wide;
      u32x4 x = {0, 0, 0, 0};
      if (c < DC) {
        if (c < d.dc) x = *reinterpret_cast<const u32x4*>(src + c);
      } else if (c - DC < d.dr) {
        x = *reinterpret_cast<const u32x4*>(src + d.dc + c - DC);
      }
      *reinterpret_cast<u32x4*>(sk + L::off(e / PR, e % PR)) = x;
    }
    __syncthreads();
    f32x4 s[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) s[i] = zero4();
#pragma unroll
    for (int t = 0; t < KS; ++t)
#pragma unroll
      for (int i = 0; i < MT; ++i) s[i] = M16<T>::mma(L::row16(sk, 16 * (MT * tw + i), 32 * t), qf[t], s[i]);
    const int lim = min(end, seen) - k0 - 16 * MT * tw;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[i][r] = 16 * i + tile_row(r) < lim ? s[i][r] * c2 : -INFINITY;
        top = fmaxf(top, s[i][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float mn = fmaxf(m, top), ref = mn == -INFINITY ? 0.f : mn, fade = fast_exp2(m - ref);
    m = mn;
    sum *= fade;
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n] *= fade;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      half p;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = fast_exp2(s[i][r] - ref);
        sum += e;
        p[r] = (T)e;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n] = M16<T>::mma4(L::col16(sk, 16 * (MT * tw + i), 16 * n), p, acc[n]);
    }
  }
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  // the TW waves of a row group: a common maximum, then sums pairwise through LDS
  if constexpr (TW > 1) {
    if (lane_id() < 16) {
      sm[wv][lane_id()] = m;
      ss[wv][lane_id()] = sum;
    }
    __syncthreads();
    const int col = lane_id() & 15;
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
        for (int n = 0; n < NT; ++n) x[(((tw - hw) * MT + rw) * NT + n) * 64 + lane_id()] = acc[n];
      }
      __syncthreads();
      if (tw < hw) {
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[n] += x[((tw * MT + rw) * NT + n) * 64 + lane_id()];
      }
    }
  }
  if (tw != 0 || row >= rows) return;
  const int64_t at = ((int64_t)b * d.splits + sp) * rows + row;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = 16 * n + tile_row(0);
    if (c < d.dc) store4(part + at * d.dc + c, acc[n]);
  }
  if (lane_id() < 16) {
    stat[2 * at] = m;
    stat[2 * at + 1] = sum;
  }
}

// o: joins the splits of 16 query tokens of a head and multiplies with the
// head's value projection, 64 value columns a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void latent_up(DecDims d, const T* __restrict__ w_kv, const float* __restrict__ part,
                                                 const float* __restrict__ stat, const int32_t* __restrict__ kv_lens,
                                                 T* __restrict__ o) {
  constexpr int V = 16 / (int)sizeof(T), LD = 512 + V, KS = 32, PARTS = sizeof(T) == 2 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) T so[PARTS][16 * LD];
  const int h = blockIdx.x, v0 = 64 * blockIdx.y, r0 = 16 * blockIdx.z, R = d.B * d.n, rows = d.n * d.H;
  {
    const int r = min(r0 + (int)(threadIdx.x >> 4), R - 1), b = r / d.n, rr = r % d.n * d.H + h;
    const int len = dec_len(d, kv_lens, b), ns = (len + d.chunk - 1) / d.chunk;
    const int64_t at = (int64_t)b * d.splits * rows + rr;
    float m = -INFINITY;
    for (int s = 0; s < ns; ++s) m = fmaxf(m, stat[2 * (at + (int64_t)s * rows)]);
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
    for (int s = 0; s < ns; ++s)
      sum += stat[2 * (at + (int64_t)s * rows) + 1] * fast_exp2(stat[2 * (at + (int64_t)s * rows)] - ref);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    for (int c = 4 * (threadIdx.x & 15); c < (d.dc + 31) / 32 * 32; c += 64) {
      f32x4 x = zero4();
      if (c < d.dc)
        for (int s = 0; s < ns; ++s) {
          const int64_t a = at + (int64_t)s * rows;
          const float w = fast_exp2(stat[2 * a] - ref) * inv;
          x += w * *reinterpret_cast<const f32x4*>(part + a * d.dc + c);
        }
      store4(&so[0][(threadIdx.x >> 4) * LD + c], x);
      if constexpr (PARTS == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] -= (float)(T)x[j];
        store4(&so[PARTS - 1][(threadIdx.x >> 4) * LD + c], x);
      }
    }
  }
  __syncthreads();
  const int vr = v0 + 16 * wave_id();
  if (vr >= d.dv) return;
  const T* w = w_kv + ((int64_t)h * (d.dn + d.dv) + d.dn + min(vr + (lane_id() & 15), d.dv - 1)) * d.dc;
  f32x4 acc = zero4();
#pragma unroll 4
  for (int k0 = 0; k0 < d.dc; k0 += KS) {
    const int k = k0 + 8 * (lane_id() >> 4);
    const typename M16<T>::frag a = k < d.dc ? ld_frag(w + k) : zero_frag<T>();
#pragma unroll
    for (int p = 0; p < PARTS; ++p) acc = M16<T>::mma(a, ld_frag(&so[p][(lane_id() & 15) * LD + k]), acc);
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

// rows a workgroup of latent_split takes, in tiles of 16
static int dec_row_tiles(const atomic_latent_decode_args* a) {
  const int rows = a->tokens * a->heads;
  return rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
}

static DecDims dec_dims(const atomic_latent_decode_args* a) {
  DecDims d{a->batch, a->tokens, a->heads, a->dn, a->dr, a->dv, a->dc, a->page, a->pages, a->table_pages,
            a->rope_rows, a->interleaved, 0, 0, 0, a->scale, {a->q_stride[0], a->q_stride[1], a->q_stride[2]}};
  const int rt = 16 * dec_row_tiles(a);
  d.groups = (d.n * d.H + rt - 1) / rt;
  // about 512 workgroups if every sequence were as long as its table
  const int64_t most = (int64_t)d.table * d.page, want = most * d.B * d.groups / 512;
  const int64_t chunk = want < 64 ? 64 : want > 2048 ? 2048 : want;
  d.chunk = (int)((chunk + 63) / 64 * 64);
  d.splits = (int)((most + d.chunk - 1) / d.chunk);
  return d;
}
static size_t up256(size_t x) { return (x + 255) / 256 * 256; }
static size_t dec_qa_bytes(const DecDims& d, int dtype) {
  return up256((size_t)d.B * d.n * d.H * (d.dc + d.dr) * (dtype == ATOMIC_BF16 ? 2 : 4));
}
static size_t dec_part_rows(const DecDims& d) { return (size_t)d.B * d.splits * d.n * d.H; }

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
  return dec_qa_bytes(d, a->dtype) + up256(dec_part_rows(d) * 8) + dec_part_rows(d) * d.dc * sizeof(float);
}

template <typename T, int DC>
static void launch_split(const DecDims& d, int mt, hipStream_t st, const T* qa, const void* cache, const int32_t* table,
                         const int32_t* kv_lens, float* part, float* stat) {
  const dim3 grid((unsigned)d.splits, (unsigned)d.groups, (unsigned)d.B);
  if (mt == 1)
    hipLaunchKernelGGL((latent_split<T, DC, 1>), grid, dim3(256), 0, st, d, qa, (const T*)cache, table, kv_lens, part,
                       stat);
  else if (mt == 2)
    hipLaunchKernelGGL((latent_split<T, DC, 2>), grid, dim3(256), 0, st, d, qa, (const T*)cache, table, kv_lens, part,
                       stat);
  else
    hipLaunchKernelGGL((latent_split<T, DC, 4>), grid, dim3(256), 0, st, d, qa, (const T*)cache, table, kv_lens, part,
                       stat);
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
    float* stat = (float*)((char*)workspace + dec_qa_bytes(d, a->dtype));
    float* part = (float*)((char*)stat + up256(dec_part_rows(d) * 8));
    const unsigned rt = (unsigned)((d.B * d.n + 15) / 16);
    int rc = L("latent_absorb", [&] {
      hipLaunchKernelGGL((latent_absorb<T>), dim3((unsigned)d.H, (unsigned)((d.dc + 63) / 64 + 1), rt), dim3(256), 0,
                         st, d, (const T*)q, (const T*)w_kv, kv_lens, cos, sin, qa);
    });
    if (rc) return rc;
    rc = L("latent_split", [&] {
      if (d.dc <= 256)
        launch_split<T, 256>(d, dec_row_tiles(a), st, qa, cache, page_table, kv_lens, part, stat);
      else
        launch_split<T, 512>(d, dec_row_tiles(a), st, qa, cache, page_table, kv_lens, part, stat);
    });
    if (rc) return rc;
    return L("latent_up", [&] {
      hipLaunchKernelGGL((latent_up<T>), dim3((unsigned)d.H, (unsigned)((d.dv + 63) / 64), rt), dim3(256), 0, st, d,
                         (const T*)w_kv, part, stat, kv_lens, (T*)o);
    });
  };
  return a->dtype == ATOMIC_BF16 ? go(bf16()) : go(float());
}
