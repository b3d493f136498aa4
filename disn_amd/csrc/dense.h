// dense.h -- what linear.hip and norm.hip share: element types, unaligned vector loads and stores, the sum over
// partial column sums.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// 16 bytes of T.  Rows start at any address that fits T (odd widths, slices), so the accesses go through memcpy with
// T's own alignment: hipcc makes one global_load/store_dwordx4 of each, which the hardware takes at any address.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
// rounds N values to T, two at a time (one conversion instruction each)
template <typename T, int N>
__device__ __forceinline__ void narrow(const float* z, T* out) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = z[i];
  } else {
    typedef __attribute__((ext_vector_type(2))) float float2v;
    typedef __attribute__((ext_vector_type(2))) T pair;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const pair p = __builtin_convertvector((float2v){z[i], z[i + 1]}, pair);
      out[i] = p[0];
      out[i + 1] = p[1];
    }
  }
}

// The first n values at p (n >= N: all, n <= 0: none), zeros behind them; nothing outside the row is read.  before: how
// many values of the row lie in front of p; with N - n of them the piece is read from so much further in front and shifted.
// (No sequence of single loads beside the wide one: hipcc merges the two into three narrow loads for every lane.)
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p, int n, int64_t before) {
  constexpr int N = Vec<T>::N;
  if (n >= N) return load_vec(p);
  const int back = N - n;
  uint64_t w[2] = {0, 0};
  if (n > 0) {
    if (back <= before) {
      __builtin_memcpy(w, p - back, 16);
      const int s = back * (8 * (int)sizeof(T));
      if (s >= 64) {
        w[0] = w[1] >> (s - 64);
        w[1] = 0;
      } else {
        w[0] = (w[0] >> s) | ((w[1] << 1) << (63 - s));
        w[1] >>= s;
      }
    } else {   // a row of fewer than N values
#pragma unroll 1
      for (int i = n - 1; i >= 0; --i) {
        uint64_t bits = 0;
        __builtin_memcpy(&bits, p + i, sizeof(T));
        w[1] = (w[1] << (8 * sizeof(T))) | (w[0] >> (64 - 8 * sizeof(T)));
        w[0] = (w[0] << (8 * sizeof(T))) | bits;
      }
    }
  }
  return __builtin_bit_cast(Vec<T>, w);
}
// what a load from `back` (< N) values further in front gave, without those values; zeros behind
template <typename T>
__device__ __forceinline__ Vec<T> shift_vec(const Vec<T>& v, int back) {
  uint64_t w[2];
  __builtin_memcpy(w, &v, 16);
  const int s = back * (8 * (int)sizeof(T));
  const uint64_t hi = w[1];
  w[0] = s >= 64 ? hi >> (s & 63) : (w[0] >> s) | ((hi << 1) << (63 - s));
  w[1] = s >= 64 ? 0 : hi >> s;
  return __builtin_bit_cast(Vec<T>, w);
}
// 16 bytes past the caches' usual order of keeping them: results are written once, and the operands around them are read
// again.  65536 x 512 x 1536 bf16 135 -> 127 us, 262144 x 64 x 512 83 -> 72; a chain of layers whose values would fit the last
// cache gains too (four of 16384 x 512 x 512: 68 -> 65).
template <typename T>
__device__ __forceinline__ void stream_vec(T* p, const Vec<T>& r) {
  typedef __attribute__((ext_vector_type(4))) uint32_t four;
  typedef four words __attribute__((aligned(2)));   // any address that fits T
  asm volatile("");   // (without the two, a branch between this store and an ordinary one becomes one ordinary store)
  __builtin_nontemporal_store(__builtin_bit_cast(words, r), (words*)p);
  asm volatile("");
}
// the first n (n >= N: all) values to p
template <typename T, bool STREAM = false>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& r, int n) {
  if (n >= Vec<T>::N) {
    if (STREAM) stream_vec(p, r);
    else __builtin_memcpy(p, &r, 16);
  } else {
    uint64_t w[2];
    __builtin_memcpy(w, &r, 16);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      __builtin_memcpy(p + i, w, sizeof(T));
      w[0] = (w[0] >> (8 * sizeof(T))) | (w[1] << (64 - 8 * sizeof(T)));
      w[1] >>= 8 * sizeof(T);
    }
  }
}

// Sum of partial column sums: out[c] = part[0][c] + part[1][c] + ... .  A workgroup takes 16 columns; its 16 groups of
// 16 threads add every 16th partial each, and the group sums are added in order (a fixed association).
// Columns [0, d) go to out0, [d, 2 d) to out1 (a layer norm's two gradients; ncols = d or 2 d), either may be null.
template <typename T>
__global__ __launch_bounds__(256) void k_sum_partials(const float* __restrict__ part, int nparts, int64_t ncols, int64_t d,
                                                      T* __restrict__ out0, T* __restrict__ out1) {
  __shared__ float lds[16][17];
  const int c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int64_t col = (int64_t)blockIdx.x * 16 + c;
  float s = 0.0f;
  if (col < ncols) {
    int p = g;
    for (; p + 15 * 16 < nparts; p += 16 * 16) {   // sixteen loads under way
      float v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = part[(size_t)(p + u * 16) * ncols + col];
#pragma unroll
      for (int u = 0; u < 16; ++u) s += v[u];
    }
    for (; p < nparts; p += 16) s += part[(size_t)p * ncols + col];
  }
  lds[g][c] = s;
  __syncthreads();
  if (g == 0 && col < ncols) {
    float t = lds[0][c];
#pragma unroll
    for (int i = 1; i < 16; ++i) t += lds[i][c];
    T* out = col < d ? out0 : out1;
    if (out) out[col < d ? col : col - d] = (T)t;
  }
}

inline bool dense_type_ok(int t) { return t == DISN_F32 || t == DISN_BF16 || t == DISN_F16; }
inline size_t dense_type_size(int t) { return t == DISN_F32 ? 4 : 2; }
inline bool dense_aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline bool dense_size_ok(int64_t v) { return v >= 0 && v <= 1 << 30; }
// a matrix argument: present, fits its type's alignment, row distance possible.  Row distances are bounded so that
// rows * ld * size stays inside 63 bits.
inline bool dense_matrix_ok(const void* p, int64_t rows, int64_t cols, int64_t ld, size_t size, bool input) {
  if (rows == 0 || cols == 0) return true;
  return p && dense_aligned(p, size) && ld <= (int64_t)1 << 31 && (ld >= cols || (input && ld == 0) || (rows == 1 && ld >= 0));
}

template <typename F>
inline int dense_dispatch(int type, F&& f) {
  if (type == DISN_F32) return f((float)0);
  if (type == DISN_BF16) return f((bf16_t)0.0f);
  return f((f16_t)0.0f);
}
