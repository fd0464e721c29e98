// Shared pieces of the latent-attention kernels: 32 x 32 MFMA fragments, the
// LDS tile layout and the host checks.
//
// Every product is arranged so that the softmax's row (a query) runs along the
// columns of an MFMA result: S^T = K Q^T gives lane l (query l % 32) the scores
// of tokens 8 (r / 4) + 4 (l / 32) + r % 4, and registers 8 s .. 8 s + 7 of it
// are, as they stand, the B operand of the next product over the 16 tokens of
// step s (its k order is the same permutation on both sides).  So probabilities
// and score gradients never leave the registers.
#pragma once
#include "common.hpp"
#include "launch.hpp"
#include "ws_tag.hpp"

namespace ah {

typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// A row's reference may lag its true maximum by this many powers of two before the
// accumulators are rescaled: p stays below 2^8, and most tiles need neither the
// maximum across lanes nor a rescale.
constexpr float kLag = 8.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// v_log_f32 flushes subnormals; the arguments here are sums of at least one 1.0
__device__ __forceinline__ float fast_log2(float x) { return __builtin_amdgcn_logf(x); }

template <typename T> struct M32;
template <> struct M32<bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
// fp32: the same eight k values a lane, as eight instructions of two k values
// (one from each half of the wave)
template <> struct M32<float> {
  typedef f32x8 frag;
  static __device__ __forceinline__ f32x16 mma(frag a, frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// Eight consecutive elements as a fragment (zeros where !ok: the padding of a width).
__device__ __forceinline__ bf16x8 ld_frag(const bf16* p) { return *reinterpret_cast<const bf16x8*>(p); }
__device__ __forceinline__ f32x8 ld_frag(const float* p) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T> __device__ __forceinline__ typename M32<T>::frag zero_frag() {
  typename M32<T>::frag z;
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = (T)0.f;
  return z;
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int j = 0; j < 16; ++j) z[j] = 0.f;
  return z;
}

// What rounding to T leaves out.
template <typename T> __device__ __forceinline__ f32x4 rounding(f32x4 x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] -= (float)(T)x[j];
  return x;
}

// A tile of rows of W elements in LDS as 16-byte pieces, piece c of row r at
// place c ^ swz(r).  With FR rows a fragment (32 or 16), the row reads (16 bytes a
// lane) and the transposed reads (8 bytes a lane) both run without bank conflicts
// (256 bytes a clock over 64 banks; measured one wave's pattern each: rows of 256
// bytes and more want all four bits, 16-row fragments in their own order; with
// only 128 bytes swizzled the row reads took twice as long).
template <typename T, int W, int FR = 32>
struct LTile {
  static constexpr int VEC = 16 / (int)sizeof(T);
  static constexpr int NC = (W / VEC + 7) / 8 * 8;
  static constexpr int ROWB = NC * 16;
  static __device__ __forceinline__ int swz(int r) {
    return NC == 8 ? (r >> 1) & 7 : FR == 16 ? r & 15 : ((r & 3) << 2) | ((r >> 2) & 3);
  }
  // (the piece's upper bits apart: they become the read's immediate offset)
  static __device__ __forceinline__ int off(int r, int c) {
    return r * ROWB + (((c & M) ^ swz(r)) << 4) + ((c & ~M) << 4);
  }
  // Row operand: lane (l % 32) holds row r0 + l % 32, elements k0 + 8 (l / 32) .. + 7.
  // `base`: the tile's LDS address plus row_base.  r0 is a multiple of 32 and k0 of 16,
  // so what differs between two reads is a constant: one exclusive-or and the immediate
  // offset.  (Addresses of their own would be kept in registers over the loop; the
  // forward spilled 20 of them, and every reload waited for the tile in flight.)
  static __device__ __forceinline__ uint32_t row_base() {
    const int l = lane_id();
    return off(l & 31, 8 / VEC * (l >> 5));
  }
  static __device__ __forceinline__ typename M32<T>::frag row(uint32_t base, int r0, int k0) {
    typedef const __attribute__((address_space(3))) char* lds_p;
    const lds_p p = (lds_p)(base ^ piece(k0 / VEC)) + r0 * ROWB + above(k0 / VEC);
    if constexpr (sizeof(T) == 2) {
      return *(const __attribute__((address_space(3))) bf16x8*)p;
    } else {
      const lds_p p1 = (lds_p)(base ^ piece(k0 / VEC + 1)) + r0 * ROWB + above(k0 / VEC);
      const f32x4 a = *(const __attribute__((address_space(3))) f32x4*)p;
      const f32x4 b = *(const __attribute__((address_space(3))) f32x4*)p1;
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  // Column operand: lane (l % 32) holds column c0 + l % 32 of the 16 rows from r0, in the order that
  // a result's registers have: rows r0 + 4 (l / 32) + j and r0 + 8 + 4 (l / 32) + j.
  // r0 is a multiple of 16 and c0 of 32; the swizzle of 8 a + 4 h + b is that of the three apart.
  static __device__ __forceinline__ uint32_t col_base() {
    const int l = lane_id(), h = l >> 5, t = l & 15;
    if constexpr (sizeof(T) == 2) {
      const int c = 16 * ((l >> 4) & 1) + 4 * (t & 3);
      return off(4 * h + (t >> 2), c / 8) + 2 * (c & 7);
    } else {
      return off(4 * h, (l & 31) / 4) + 4 * (l & 3);
    }
  }
  static __device__ __forceinline__ typename M32<T>::frag col(uint32_t base, int r0, int c0) {
    typedef const __attribute__((address_space(3))) char* lds_p;
    const int c = c0 / VEC;
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) bf16x4* v4_p;
      const lds_p p = (lds_p)(base ^ piece(c)) + r0 * ROWB + above(c);
      const lds_p p8 = (lds_p)(base ^ piece(c) ^ (swz(8) << 4)) + (r0 + 8) * ROWB + above(c);
      const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((v4_p)p);
      const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((v4_p)p8);
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      f32x8 z;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 8 * (j >> 2) + (j & 3);
        const lds_p p = (lds_p)(base ^ piece(c) ^ (swz(r) << 4)) + (r0 + r) * ROWB + above(c);
        z[j] = *(const __attribute__((address_space(3))) float*)p;
      }
      return z;
    }
  }
  static constexpr int M = NC == 8 ? 7 : 15;
  static __device__ __forceinline__ uint32_t piece(int c) { return (c & M) << 4; }
  static __device__ __forceinline__ int above(int c) { return (c & ~M) << 4; }
};

// use(i, load(i)) for i in [0, N), each use one MFMA, in groups of G, with its
// operand read from LDS `LA` groups ahead (left alone, the compiler reads each
// fragment right before its MFMA and waits for it there).  work(i) is other work
// done at slot i; VN > 0 spreads a group's vector instructions over its MFMAs, VN
// after each, where they run while the matrix pipe is busy.  A use may be MF MFMAs.
template <int N, int G, int LA, int VN, typename F, int MF = 1, typename L, typename U, typename K>
__device__ __forceinline__ void in_groups(L&& load, U&& use, K&& work) {
  F f[LA + 1][G];
  static_for<(LA * G < N ? LA * G : N)>([&](auto j) { f[j.value / G][j.value % G] = load(j.value); });
  __builtin_amdgcn_sched_barrier(0);
  static_for<(N + G - 1) / G>([&](auto gr) {
    constexpr int g = decltype(gr)::value;
    static_for<G>([&](auto j) {
      constexpr int at = (g + LA) * G + decltype(j)::value;
      if constexpr (at < N) f[(g + LA) % (LA + 1)][j.value] = load(at);
    });
    if constexpr (VN == 0) __builtin_amdgcn_sched_barrier(0);
    static_for<G>([&](auto j) {
      if constexpr (g * G + decltype(j)::value < N) work(g * G + j.value);
    });
    static_for<G>([&](auto j) {
      if constexpr (g * G + decltype(j)::value < N) use(g * G + j.value, f[g % (LA + 1)][j.value]);
    });
    if constexpr (VN > 0) {
      __builtin_amdgcn_sched_group_barrier(0x100, 4 * G, 0);  // LDS reads
      static_for<G * MF>([&](auto) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // MFMA
        __builtin_amdgcn_sched_group_barrier(0x002, VN, 0);  // vector
      });
    }
    __builtin_amdgcn_sched_barrier(0);
  });
}
template <int N, int G, typename F, typename L, typename U>
__device__ __forceinline__ void in_groups(L&& load, U&& use) {
  in_groups<N, G, 1, 0, F>(load, use, [](int) {});
}

// Rows of a matrix (W elements, `width` of them real) straight to an LTile of ROWS
// rows, NW waves taking 1 KB each in turn: wave w's i-th load covers the rows
// RPI (w + NW i) .. + RPI - 1.  Rows past `last` are zeros (their products are masked,
// and what lies there is never read); the padding of the width reads the row's first
// piece (the other operand is zero there, or the product's column is not stored).
//
// A load is one instruction and no vector arithmetic, to be spread over the MFMAs
// of a tile: a CU takes 64 bytes a clock on this path, so a tile's 40 KB sent for at
// once hold every wave up for 600 to 1000 clocks.
constexpr int64_t kMostRowBytes = 1 << 25;  // a tile's byte offsets have to fit 31 bits
template <typename T, int W, int ROWS, int NW>
struct RowDma {
  typedef LTile<T, W> L;
  static constexpr int RPI = 64 / L::NC, N = ROWS / RPI / NW, STEP = NW * RPI;
  static constexpr int NZ = STEP >= 16 ? 1 : 16 / STEP;  // the swizzle repeats every 16 rows
  static_assert(RPI * L::NC == 64 && N * STEP == ROWS && (STEP >= 16 || 16 % STEP == 0), "whole loads");
  uint64_t base;      // the first row aimed at
  int left;           // rows from it to the last
  uint32_t ld, wide;  // bytes between rows, bytes of a row
  uint32_t at[NZ];    // this lane's byte in the first load
  int w;              // this wave among the NW
  buffer_t d;
  __device__ __forceinline__ void init(const T* p, int64_t stride, int width) {
    w = NW == 1 ? 0 : wave_id();
    base = (uint64_t)p;
    ld = (uint32_t)(stride * (int64_t)sizeof(T));
    wide = width * (uint32_t)sizeof(T);
    const int r0 = RPI * w + lane_id() / L::NC;
#pragma unroll
    for (int z = 0; z < NZ; ++z) {
      const int c = (lane_id() % L::NC) ^ L::swz(r0 + z * STEP);
      at[z] = r0 * ld + (c * L::VEC < width ? 16 * c : 0);
    }
  }
  // the rows k0 .. last are next, a tile at a time; zeros past them
  __device__ __forceinline__ void start(int k0, int last) {
    ld = __builtin_amdgcn_readfirstlane(ld);
    base += (uint64_t)k0 * ld;
    base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(base >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)base);
    left = __builtin_amdgcn_readfirstlane(last - k0 + 1);
  }
  __device__ __forceinline__ void aim() {
    d = buffer_of(base, left > 0 ? (uint32_t)(min(left, ROWS) - 1) * ld + wide : 0);
    base += ROWS * (uint64_t)ld;
    left -= ROWS;
  }
  // the same for one tile by itself, without `start`
  __device__ __forceinline__ void aim_at(int k0, int last) {
    d = buffer_of(base + (uint64_t)k0 * ld, k0 <= last ? (uint32_t)min(last - k0, ROWS - 1) * ld + wide : 0);
  }
  // this wave's i-th load; `dst`: the tile's LDS address
  __device__ __forceinline__ void load(int i, uint32_t dst) const {
    dma16_buf(d, at[i % NZ], (uint32_t)(i * STEP) * ld, dst + 1024 * (w + NW * i));
  }
};
// Three of them one after the other: the tiles of a stage.
template <typename A, typename B, typename C>
struct StageDma {
  A a;
  B b;
  C c;
  uint32_t ob, oc;  // where the second and the third tile lie behind the first
  static constexpr int N = A::N + B::N + C::N;
  __device__ __forceinline__ void start(int k0, int last) {
    a.start(k0, last);
    b.start(k0, last);
    c.start(k0, last);
  }
  __device__ __forceinline__ void aim() {
    a.aim();
    b.aim();
    c.aim();
  }
  __device__ __forceinline__ void aim_at(int k0, int last) {
    a.aim_at(k0, last);
    b.aim_at(k0, last);
    c.aim_at(k0, last);
  }
  __device__ __forceinline__ void load(int i, uint32_t dst) const {
    if (i < A::N) a.load(i, dst);
    else if (i < A::N + B::N) b.load(i - A::N, dst + ob);
    else c.load(i - A::N - B::N, dst + oc);
  }
  // the loads that belong to slot j of `slots`
  __device__ __forceinline__ void at_slot(int j, int slots, uint32_t dst) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * slots / N == j) load(i, dst);
  }
  __device__ __forceinline__ void all(uint32_t dst) const {
#pragma unroll
    for (int i = 0; i < N; ++i) load(i, dst);
  }
};

inline int latent_widths_check(int dn, int dr, int dtype) {
  if (dtype != ATOMIC_F32 && dtype != ATOMIC_BF16) return ATOMIC_ERR_DTYPE;
  if (dn < 8 || dn > 128 || dn % 8 || dr < 8 || dr > 64 || dr % 8) return ATOMIC_ERR_SHAPE;
  return ATOMIC_OK;
}
inline bool whole_pieces(std::initializer_list<int64_t> strides, int dtype) {
  const int64_t v = dtype == ATOMIC_BF16 ? 8 : 4;
  for (int64_t s : strides)
    if (s < 0 || s % v || s > INT64_MAX / 16) return false;
  return true;
}

}  // namespace ah
