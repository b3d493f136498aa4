// linear.hip -- the dense layer y = act(x W + b) + r and its gradients (include/disn.h).
//
// Forward and both gradients are one product C(i, j) = sum over r of A(i, r) B(j, r) with different operands:
//   y   i = row, j = output, r = input     A = x                    B = W
//   dx  i = row, j = input,  r = output    A = dz                   B = W
//   dW  r = row                            A = x, B = dz ([k][n]) or A = dz, B = x ([n][k])
// An operand lies "along" r (its r values are contiguous) or "across" (its i values are, rows of r).
//
// The kernels that compute it, chosen by size (plan() below):
//   k_tile16, k_tile32  large products: 128- or 256-wide tiles through LDS on the matrix cores
//   k_small  products of some microseconds: no LDS tiles, the waves of a workgroup share the sum
//   k_rows_* at most 4 rows times a large matrix: W streams past at memory speed
//   k_outer  sums of up to 8 products: C is what takes time to write
//   k_thin   long sums for a C of up to 8 rows or columns: the wider operand is what takes time to read
#include "dense.h"
#define EDGE_QUAL __device__ __forceinline__
#include "tile_edge.h"

#include <atomic>
#include <type_traits>

namespace {

typedef __attribute__((ext_vector_type(16))) float floatx16;
typedef __attribute__((ext_vector_type(4))) float floatx4;
typedef __attribute__((ext_vector_type(4))) short shortx4;
typedef __attribute__((ext_vector_type(8))) short shortx8;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
typedef __attribute__((address_space(3))) char lds_char;

// ---- activations ------------------------------------------------------------------------------------------------
// The normal distribution's upper tail Q(u) = P(u) exp(-u^2 / 2) for u >= 0, P a polynomial in 1 / (1 + 0.26 u) fitted to
// erfc(u / sqrt 2) exp(u^2 / 2) / 2 (least squares, reweighted towards the smallest largest error): |error| < 2.2e-7 in
// float32 arithmetic.  A third of the instructions of erff, whose two branches both run in most waves.
// tail returns Q, e = exp(-u^2 / 2).
__device__ __forceinline__ float normal_tail(float u, float& e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.26f, u, 1.0f));
  float p = fmaf(-0.07304021f, t, 0.22896615f);
  p = fmaf(p, t, -0.10594359f);
  p = fmaf(p, t, 0.16563688f);
  p = fmaf(p, t, 0.07380697f);
  p = fmaf(p, t, 0.10704367f);
  p = fmaf(p, t, 0.10353009f);
  e = __builtin_amdgcn_exp2f(u * u * -0.72134752f);
  return p * t * e;
}
// The normal distribution's integral from below to z; e = exp(-z^2 / 2).  Half a step of a 16-bit result is far above the error
// of the tail.  In float32 it is up to four steps of 1/2, so next to 0 it is 1/2 + z R(z^2), R a polynomial fitted to the integral's
// own series on z^2 < 1.5 (least squares, reweighted; 8e-9 of the value): gelu within 1.3e-7 of itself for z > -0.5, as erff
// gives it (5e-7 from the tail).
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float q = normal_tail(fabsf(z), e), p = z > 0.0f ? 1.0f - q : q;
  if constexpr (sizeof(T) == 2) return p;
  const float s = z * z;
  float r = fmaf(-6.8982026e-6f, s, 1.1134986e-4f);
  r = fmaf(r, s, -1.1842096e-3f);
  r = fmaf(r, s, 9.972464e-3f);
  r = fmaf(r, s, -6.649024e-2f);
  r = fmaf(r, s, 0.3989423f);
  return s < 1.5f ? fmaf(z, r, 0.5f) : p;
}
// 1 / (1 + exp(-z)).  The product with log2 e is rounded, which is |z| 2^-24 of the exponential: nothing beside half a step of a 16-bit
// result, but 1e-6 of silu at -10 in float32, where what the product and its constant lost is made up for (not where the
// exponential is infinite or 0).
template <typename T>
__device__ __forceinline__ float logistic(float z) {
  const float t = z * -1.44269504f;
  float p = __builtin_amdgcn_exp2f(t);
  if constexpr (sizeof(T) == 4) {
    const float lost = fmaf(z, -1.92596299e-8f, fmaf(z, -1.44269504f, -t));
    p = fabsf(z) < 88.0f ? fmaf(p, lost * 0.69314718f, p) : p;
  }
  return __builtin_amdgcn_rcpf(1.0f + p);
}

// T: the type of the result
template <typename T>
__device__ __forceinline__ float activate(float z, int act) {
  float e;
  switch (act) {
    case DISN_ACT_RELU: return z < 0.0f ? 0.0f : z;   // NaN stays
    case DISN_ACT_GELU: return z * normal_cdf<T>(z, e);
    case DISN_ACT_SILU: return z * logistic<T>(z);
    default: return z;
  }
}
template <typename T, int N>
__device__ __forceinline__ void activate_all(float (&z)[N], int act) {
  switch (act) {   // one branch for all of them
    case DISN_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = activate<T>(z[i], DISN_ACT_RELU);
      break;
    case DISN_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = activate<T>(z[i], DISN_ACT_GELU);
      break;
    case DISN_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = activate<T>(z[i], DISN_ACT_SILU);
      break;
  }
}
// dy act'(z)
template <typename T>
__device__ __forceinline__ float gated(float dy, float z, int act) {
  float e;
  switch (act) {
    case DISN_ACT_RELU: return z > 0.0f ? dy : z <= 0.0f ? 0.0f : z;   // a choice: closed, it passes nothing of an infinity either
    case DISN_ACT_GELU: {
      const float p = normal_cdf<T>(z, e);
      return dy * fmaf(z * 0.39894228f, e, p);
    }
    case DISN_ACT_SILU: {
      const float s = logistic<T>(z);
      return dy * (s * fmaf(z, 1.0f - s, 1.0f));
    }
    default: return dy;
  }
}

template <typename T, int N, typename Z>
__device__ __forceinline__ void gate_all(float (&dy)[N], const Z& z, int act) {
  if (act == DISN_ACT_RELU) {   // one branch for all of them
#pragma unroll
    for (int i = 0; i < N; ++i) dy[i] = gated<T>(dy[i], (float)z[i], DISN_ACT_RELU);
  } else if (act == DISN_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) dy[i] = gated<T>(dy[i], (float)z[i], DISN_ACT_GELU);
  } else if (act == DISN_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) dy[i] = gated<T>(dy[i], (float)z[i], DISN_ACT_SILU);
  }
}

// ---- what becomes of a finished sum ------------------------------------------------------------------------------
struct Epilogue {
  const void *bias, *residual;
  void *pre, *out;
  int64_t ldr, ldp, ldo;
  int act, stream;   // stream: out and pre are stored past the caches (streams())
};
template <typename T>
__device__ __forceinline__ void finish_one(const Epilogue& e, int64_t row, int col, float z) {
  if (e.bias) z += (float)((const T*)e.bias)[col];
  if (e.pre) ((T*)e.pre)[row * e.ldp + col] = (T)z;
  float y = activate<T>(z, e.act);
  if (e.residual) y += (float)((const T*)e.residual)[row * e.ldr + col];
  ((T*)e.out)[row * e.ldo + col] = (T)y;
}
// n (>= 1) of Vec<T>::N values to out and pre (if wanted); the bias and the residual (anything where there is none) have been
// read before
template <typename T>
__device__ __forceinline__ void finish_vec(const Epilogue& e, T* out, T* pre, float (&z)[Vec<T>::N], int n, const Vec<T>& bias,
                                           const Vec<T>& residual) {
  constexpr int N = Vec<T>::N;
  if (e.bias) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] += (float)bias.v[i];
  }
  Vec<T> o;
  if (e.pre) {
    narrow<T, N>(z, o.v);
    if (e.stream) store_vec<T, true>(pre, o, n);
    else store_vec(pre, o, n);
  }
  activate_all<T>(z, e.act);
  if (e.residual) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] += (float)residual.v[i];
  }
  narrow<T, N>(z, o.v);
  if (e.stream) store_vec<T, true>(out, o, n);
  else store_vec(out, o, n);
}
template <typename T>
__device__ __forceinline__ Vec<T> bias_vec(const Epilogue& e, int col, int n) {
  return e.bias && n > 0 ? load_vec((const T*)e.bias + col, n, col) : Vec<T>{};
}
template <typename T>
__device__ __forceinline__ Vec<T> residual_vec(const Epilogue& e, int64_t row, int col, int n) {
  return e.residual && n > 0 ? load_vec((const T*)e.residual + row * e.ldr + col, n, col) : Vec<T>{};
}

// Sums the partial products of a split r (0 of them: an empty sum) and finishes them.  A thread takes 16 bytes of the
// result; with few results and many parts, G threads share a result's parts (every G-th each, the G sums added in order):
// one thread after another part by part took 15 us for the 64 parts of 4096 results, now 4.  21 parts of 1536 x 512 in 12.6 us
// (5.2 TB/s).
template <typename T, int G>
__global__ __launch_bounds__(256) void k_finish(const float* __restrict__ part, int nparts, int64_t M, int N, Epilogue e) {
  constexpr int V = Vec<T>::N, C = 256 / G;
  __shared__ float lds[G > 1 ? G : 1][G > 1 ? C * V : 1];
  const int64_t per_row = (N + V - 1) / V, total = M * per_row;
  const int g = threadIdx.x / C, c = threadIdx.x % C;
  for (int64_t t0 = (int64_t)blockIdx.x * C; t0 < total; t0 += (int64_t)gridDim.x * C) {
    const int64_t t = t0 + c < total ? t0 + c : total - 1, row = t / per_row;
    const int col = (int)(t - row * per_row) * V, n = N - col;
    const Vec<T> bias = bias_vec<T>(e, col, n), residual = residual_vec<T>(e, row, col, n);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = 0.0f;
    const float* s = part + (size_t)row * N + col;
    const size_t stride = (size_t)M * N;
    if (n >= V) {
#pragma unroll 4
      for (int p = g; p < nparts; p += G) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          const Vec<float> v = load_vec(s + p * stride + i);
#pragma unroll
          for (int q = 0; q < 4; ++q) z[i + q] += v.v[q];
        }
      }
    } else {
      for (int p = g; p < nparts; p += G)
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] += i < n ? s[p * stride + i] : 0.0f;
    }
    if constexpr (G > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) lds[g][c * V + i] = z[i];
      __syncthreads();
      if (g) continue;
#pragma unroll
      for (int i = 0; i < V; ++i)
        for (int k = 1; k < G; ++k) z[i] += lds[k][c * V + i];
    }
    if (t0 + c < total) finish_vec<T>(e, (T*)e.out + row * e.ldo + col, (T*)e.pre + row * e.ldp + col, z, n, bias, residual);
  }
}

// ---- tiles: what both kernels share ---------------------------------------------------------------------------------
struct TileArgs {
  const void *A, *B;
  int64_t lda, ldb;
  int M, N;
  int64_t K, per;          // r values in all and per split (a multiple of KT)
  int mt, nt, splits;
  float* part;             // [splits][M][N], splits > 1
  Epilogue e;
};

constexpr int tile_stride(int NB) { return NB * 32 + 4; }   // floats between the turned rows

// The end of a tile: a wave's MB x NB sums (i from iw, j from jw on) become partial products or finished values.
// Finishing goes through LDS (the stages' buffers, which the caller's waves have stopped reading once they meet here),
// 32 rows at a time, so that a lane finishes 16 bytes of one row.
// Lane's place in a 32 x 32 tile of C: j = l & 31, i = (g & 3) + 8 (g >> 2) + 4 (l >> 5).
template <typename T, int MB, int NB, int WAVES>
__device__ __forceinline__ void tile_end(const TileArgs& a, int split, int iw, int jw, const floatx16 (&acc)[MB][NB], float* lds) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, cj = lane & 31, ci = 4 * (lane >> 5);
  if (a.splits > 1) {
    float* part = a.part + (size_t)split * a.M * a.N;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 16; ++g) {
          const int i = iw + m * 32 + ci + (g & 3) + 8 * (g >> 2), j = jw + n * 32 + cj;
          if (i < a.M && j < a.N) part[(size_t)i * a.N + j] = acc[m][n][g];
        }
    return;
  }
  // Memory operations of a wave end in order, so a wait for a load is a wait for the stores before it: the bias is read
  // once, the residual of two pieces before the two in front of them are stored.  The loops stay loops: unrolled, they are 80 KB of code.
  constexpr int W = NB * 32, V = Vec<T>::N, STRIDE = tile_stride(NB), Q = 32 * W / V / 64, STEP = 64 / (W / V);
  const int c = lane % (W / V) * V, j = jw + c, n_j = a.N - j, r0 = lane / (W / V);
  const Vec<T> bias = bias_vec<T>(a.e, j, n_j);
  const int i_end = min(a.M, iw + MB * 32);
  // Inside the matrix and with nothing but a bias and a relu, a piece is some thirty instructions instead of a hundred; the
  // general one costs 20 us of 150 where 65536 x 1536 results follow sums of 512.
  const bool plain = iw + MB * 32 <= a.M && jw + W <= a.N && !a.e.pre && !a.e.residual && a.e.act <= DISN_ACT_RELU;
  int i = iw + r0;   // the row of the piece to come
  T* out = (T*)a.e.out + i * a.e.ldo + j;
  T* pre = (T*)a.e.pre + i * a.e.ldp + j;
  const T* from = (const T*)a.e.residual + i * a.e.ldr + j;
  const int64_t out_step = STEP * a.e.ldo, pre_step = STEP * a.e.ldp, from_step = STEP * a.e.ldr;
  Vec<T> res[2] = {};
  auto read_residual = [&](int u, int row) {
    if (a.e.residual && row < i_end && n_j > 0) res[u] = load_vec(from, n_j, j);
    from += from_step;
  };
  read_residual(0, i);
  read_residual(1, i + STEP);
  __syncthreads();
  float* mine = lds + wave * (32 * STRIDE);
  const float* my_row = mine + r0 * STRIDE + c;
#pragma unroll 1
  for (int mm = 0; mm < MB; ++mm) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int m = 0; m < MB; ++m)
      if (m == mm) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int g = 0; g < 16; ++g) mine[(ci + (g & 3) + 8 * (g >> 2)) * STRIDE + n * 32 + cj] = acc[m][n][g];
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (plain) {
      const bool relu = a.e.act == DISN_ACT_RELU;
#pragma unroll 2
      for (int q = 0; q < Q; ++q) {
        float z[V];
        __builtin_memcpy(z, __builtin_assume_aligned(my_row + q * STEP * STRIDE, 16), sizeof z);
        if (a.e.bias) {
#pragma unroll
          for (int i = 0; i < V; ++i) z[i] += (float)bias.v[i];
        }
        if (relu) {
#pragma unroll
          for (int i = 0; i < V; ++i) z[i] = activate<T>(z[i], DISN_ACT_RELU);
        }
        Vec<T> o;
        narrow<T, V>(z, o.v);
        if (a.e.stream) stream_vec(out, o);
        else __builtin_memcpy(out, &o, 16);
        out += out_step;
      }
      continue;
    }
#pragma unroll 1
    for (int q = 0; q < Q; q += 2) {   // two pieces at a time
      float z[2][V];
      Vec<T> now[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        __builtin_memcpy(z[u], __builtin_assume_aligned(my_row + (q + u) * STEP * STRIDE, 16), sizeof z[u]);
        now[u] = res[u];
        read_residual(u, i + (u + 2) * STEP);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (i < i_end && n_j > 0) finish_vec<T>(a.e, out, pre, z[u], n_j, bias, now[u]);
        i += STEP, out += out_step, pre += pre_step;
      }
    }
  }
}

// a workgroup's tile: the workgroups go to the 8 XCDs in turn; consecutive tiles share operands, so each XCD (own
// L2) takes a run of them
struct TilePlace {
  int i0, j0, split;
};
__device__ __forceinline__ TilePlace tile_place(const TileArgs& a, int block, int BM, int BN) {
  const int total = a.mt * a.nt * a.splits, run = total >> 3, rest = total & 7, xcd = block & 7;
  int id = (block >> 3) + xcd * run + (xcd < rest ? xcd : rest);
  const int tn = id % a.nt;
  id /= a.nt;
  return {id % a.mt * BM, tn * BN, id / a.mt};
}

// ---- k_tile32 --------------------------------------------------------------------------------------------------------
// A workgroup computes a BM x BN tile of C, r in stages of KT.  The stage after the next is on its way from memory to
// registers while the next lies in one LDS buffer and the waves multiply the present one from the other: one barrier a
// stage.  Waves are WM x WN; each has MB x NB tiles of v_mfma_f32_32x32x16.  Bound by the matrix cores: 100000 x 1984 x 512
// 940 us, 4096^3 605 us (227 TFLOP/s; an fp32 library product on the fp32 matrix instructions 138).
//
// An fp32 value is cut into three bf16 terms x = h + m + l (each the rounded
// rest of the one before; 8 + 8 + 8 bits hold fp32's 24, so the sum is exact), and the six products
// hh, hm, mh, mm, hl, lh are accumulated in fp32; what is left out (ml, lm, ll) is below 2^-24 of a product, as an
// FMA's rounding is.  Six bf16 MFMAs take 6/16 of the time of one fp32 MFMA of the same size.  Infinities,
// NaN and intermediate overflow cannot be cut; a tile whose sums are not all finite is computed again by fp32 MFMAs.
// Neither can values below 2^-109, whose last term's bits lie below bf16's smallest; a tile that met one (an or over the
// last terms: an instruction for two values, under 1 % of the time) looks whether its sums are small enough to notice, and is computed again if so.
//
// LDS: an operand along r as [8 r][i][16 bytes] (half a fragment is 512 bytes in one piece; 128 bytes between the 8-r
// blocks put the lanes that store a row on different banks); an operand across r as [r][i] with 64 bytes between rows,
// read through ds_read_b64_tr_b16, which hands each lane 4 r values of its i.
constexpr int KT32 = 16, PLANES = 3;

template <typename T>
__device__ __forceinline__ floatx16 mfma(shortx8 a, shortx8 b, floatx16 c) {
  if constexpr (__is_same(T, f16_t))
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <bool ACROSS, int ROWS, int THREADS, int DEPTH>
struct Operand {
  static constexpr int KT = KT32, P = PLANES, V = Vec<float>::N;
  static constexpr int PER_LINE = (ACROSS ? ROWS : KT) / V;    // 16-byte pieces in a contiguous run
  static constexpr int Q = ROWS * KT / V / THREADS;            // pieces a thread moves per stage
  static constexpr int LINE = ROWS * 2 + 64;                   // bytes of one r (across)
  static constexpr int BLOCK = ROWS * 16 + 128;                // bytes of 8 r (along)
  static constexpr int PLANE = ACROSS ? KT * LINE : KT / 8 * BLOCK;
  static constexpr int BYTES = PLANE * P;
  static_assert(Q * THREADS * V == ROWS * KT, "pieces");

  const float* ptr[Q];
  int64_t ld;
  int left;          // i values in the tile
  int first;         // the stage's first value in its row
  int lines;         // i values in the matrix
  int back[ACROSS ? Q : 1];   // how far in front a piece is read in whole stages (inside() lines)
  Vec<float> reg[DEPTH][Q];   // stages under way

  __device__ __forceinline__ void init(const float* p, int64_t ld_, int i0, int n_i, int64_t k0) {
    ld = ld_;
    left = n_i - i0;
    first = ACROSS ? i0 : (int)k0;
    lines = n_i;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int t = threadIdx.x + q * THREADS, line = t / PER_LINE, c = t % PER_LINE * V;
      // places outside the matrix read its nearest line or the tile's first piece instead: they only reach sums nobody stores
      if (ACROSS) {
        const EdgePiece e = edge_piece(c, left, V);
        back[q] = e.back;
        ptr[q] = p + (k0 + line) * ld + i0 + e.at;
      } else {
        ptr[q] = p + (int64_t)(i0 + (line < left ? line : left - 1)) * ld + k0 + c;
      }
    }
  }
  // whether whole stages need no ends to be cut
  __device__ __forceinline__ bool inside() const { return !ACROSS || lines >= V; }
  // the next stage, of which `have` (>= 1) r values exist, into reg[slot]; zeros behind them
  template <bool WHOLE>
  __device__ __forceinline__ void fetch(int slot, int have) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int t = threadIdx.x + q * THREADS, line = t / PER_LINE, c = t % PER_LINE * V;
      if (WHOLE && (!ACROSS || left >= ROWS)) {
        reg[slot][q] = load_vec(ptr[q]);
      } else if (WHOLE) {   // the last columns: read further in front, and shifted when they are stored
        reg[slot][q] = load_vec(ptr[q] - back[q]);
      } else if (ACROSS)
        reg[slot][q] = load_vec(ptr[q] - (line < have ? 0 : line * ld), line < have ? (c < left ? left - c : left) : 0, first + (c < left ? c : 0));
      else
        reg[slot][q] = load_vec(ptr[q] - (c < have ? 0 : c), have - c, first + c);
      ptr[q] += ACROSS ? KT * ld : KT;
    }
    if (!ACROSS) first += KT;
  }
  // lost: the bits of every last term are or-ed into it; below 2^-109 some lie in its lower half, which bf16 cannot hold
  __device__ __forceinline__ void store(char* lds, int slot, bool shifted, uint32_t& lost) const {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int t = threadIdx.x + q * THREADS, line = t / PER_LINE, c = t % PER_LINE * V;
      char* dst = lds + (ACROSS ? line * LINE + c * 2 : (c >> 3) * BLOCK + line * 16 + (c & 7) * 2);
      float rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) rest[i] = reg[slot][q].v[i];
      if (ACROSS && shifted) {
        const int b = back[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) rest[i] = b & 2 ? (i < 2 ? rest[i + 2] : 0.0f) : rest[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) rest[i] = b & 1 ? (i < 3 ? rest[i + 1] : 0.0f) : rest[i];
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        // (a bf16 is the upper half of a float; widened as values, hipcc converts every value a second time)
        uint32_t term[2];
        narrow<bf16_t, 4>(rest, (bf16_t*)term);
        if (p + 1 < P) {
#pragma unroll
          for (int i = 0; i < 4; ++i) rest[i] -= __builtin_bit_cast(float, i & 1 ? term[i / 2] & 0xffff0000u : term[i / 2] << 16);
        }
        __builtin_memcpy(__builtin_assume_aligned(dst + p * PLANE, 8), term, 8);
        if (p + 2 == P) {
#pragma unroll
          for (int i = 0; i < 4; ++i) lost |= __builtin_bit_cast(uint32_t, rest[i]);
        }
      }
    }
  }
  // fragment of 32 i values from i, 16 r values from 16 s: lane (l & 31) holds i + (l & 31), r = 8 (l >> 5) + 0..7
  static __device__ __forceinline__ shortx8 fragment(const char* lds, int plane, int i, int s) {
    const int lane = threadIdx.x & 63;
    if constexpr (ACROSS) {
      // a group of 16 lanes reads 4 r x 16 i: lane q supplies r = q >> 2, i = 4 (q & 3), and gets i = q of all four
      const int q = lane & 15;
      const char* p = lds + plane * PLANE + (16 * s + 8 * (lane >> 5) + (q >> 2)) * LINE + (i + (lane & 16) + 4 * (q & 3)) * 2;
      const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(p));
      const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(p + 4 * LINE));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const char* p = lds + plane * PLANE + (2 * s + (lane >> 5)) * BLOCK + (i + (lane & 31)) * 16;
      return *(const shortx8*)p;
    }
  }
};

// Over n (<= WIDTH) lines' r values k0 .. k0 + have - 1: the largest absolute value, for every thread, and 1 in live[] for every line
// that holds anything but zeros (0 there before; complete behind the caller's next barrier).  lds: a float a wave
template <bool ACROSS, int WIDTH, int THREADS>
__device__ __forceinline__ float panel_max(const float* p, int64_t ld, int line, int n, int64_t k0, int have, float* lds, uint8_t* live) {
  p += ACROSS ? k0 * ld + line : line * ld + k0;
  // 16 bytes a thread of a run of contiguous values; the last piece of a run lies over the one before it
  constexpr int PER = ACROSS ? WIDTH / 4 : 64;
  const int run = ACROSS ? n : have, runs = ACROSS ? have : n;
  float most = 0.0f;
  for (int c0 = 0; c0 < run; c0 += PER * 4) {
    const int c = c0 + (int)threadIdx.x % PER * 4, at = min(c, max(run - 4, 0));
    float column[4] = {0, 0, 0, 0};   // (ACROSS) the largest of each of the four lines
#pragma unroll 8
    for (int t = threadIdx.x / PER; t < runs; t += THREADS / PER) {
      Vec<float> v;
      if (run >= 4) v = load_vec(p + t * ld + at);
      else v = load_vec(p + t * ld, run, 0);
      if (ACROSS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) column[i] = fmaxf(column[i], fabsf(v.v[i]));
      } else {
        const float here = fmaxf(fmaxf(fabsf(v.v[0]), fabsf(v.v[1])), fmaxf(fabsf(v.v[2]), fabsf(v.v[3])));
        if (here > 0.0f) live[t] = 1;
        most = fmaxf(most, here);
      }
    }
    if (ACROSS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (column[i] > 0.0f) live[at + i] = 1;
        most = fmaxf(most, column[i]);
      }
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) most = fmaxf(most, __shfl_xor(most, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = most;
  __syncthreads();
  for (int w = 0; w < THREADS / 64; ++w) most = fmaxf(most, lds[w]);
  return most;
}

// r = r0 .. r0 + 3 (those below K) of line i (clamped to the matrix by the caller)
template <typename T, bool ACROSS, bool FULL>
__device__ __forceinline__ floatx4 load_4r(const void* p_, int64_t ld, int i, int r0, int K) {
  const T* p = (const T*)p_;
  floatx4 v;
  if constexpr (!ACROSS && FULL) {
    T t[4];
    __builtin_memcpy(t, p + i * ld + r0, sizeof t);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = FULL || r0 + e < K;
      const int r = in ? r0 + e : 0;
      const float x = (float)p[ACROSS ? r * ld + i : i * ld + r];
      v[e] = in ? x : 0.0f;
    }
  }
  return v;
}

// a wave's sums by fp32 matrix instructions on operands straight from memory, 8 r values a step
template <bool A_ACROSS, bool B_ACROSS, int MB, int NB>
__device__ __forceinline__ void fp32_sums(const TileArgs& a, int iw, int jw, int64_t k0, int have, floatx16 (&acc)[MB][NB]) {
  const int idx = threadIdx.x & 31, half = 4 * ((threadIdx.x & 63) >> 5);
  const float* pa = (const float*)a.A + (A_ACROSS ? k0 * a.lda : k0);
  const float* pb = (const float*)a.B + (B_ACROSS ? k0 * a.ldb : k0);
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int g = 0; g < 16; ++g) acc[m][n][g] = 0.0f;
  auto step = [&](int r, auto full) {
    constexpr bool FULL = decltype(full)::value;
    floatx4 va[MB], vb[NB];
#pragma unroll
    for (int m = 0; m < MB; ++m) va[m] = load_4r<float, A_ACROSS, FULL>(pa, a.lda, min(iw + m * 32 + idx, a.M - 1), r + half, have);
#pragma unroll
    for (int n = 0; n < NB; ++n) vb[n] = load_4r<float, B_ACROSS, FULL>(pb, a.ldb, min(jw + n * 32 + idx, a.N - 1), r + half, have);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(va[m][e], vb[n][e], acc[m][n], 0, 0, 0);
  };
  int r = 0;
#pragma unroll 1
  for (; r + 8 <= have; r += 8) step(r, std::true_type());
  if (r < have) step(r, std::false_type());
}

template <bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN, int DEPTH>
__device__ __forceinline__ void tile32(const TileArgs& a, int block, char* lds) {
  constexpr int THREADS = WM * WN * 64, MB = BM / WM / 32, NB = BN / WN / 32, KT = KT32, P = PLANES;
  typedef Operand<A_ACROSS, BM, THREADS, DEPTH> OpA;
  typedef Operand<B_ACROSS, BN, THREADS, DEPTH> OpB;
  constexpr int BUF = OpA::BYTES + OpB::BYTES;
  const TilePlace at = tile_place(a, block, BM, BN);
  const int i0 = at.i0, j0 = at.j0, split = at.split;
  const int64_t k0 = split * a.per;
  const int have = (int)(a.K - k0 < a.per ? a.K - k0 : a.per), stages = (have + KT - 1) / KT;
  const int wave = threadIdx.x >> 6;
  const int wi = wave / WN * (MB * 32), wj = wave % WN * (NB * 32);

  floatx16 acc[MB][NB];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int g = 0; g < 16; ++g) acc[m][n][g] = 0.0f;

  OpA A;
  OpB B;
  uint32_t lost = 0;
  A.init((const float*)a.A, a.lda, i0, a.M, k0);
  B.init((const float*)a.B, a.ldb, j0, a.N, k0);
  auto multiply = [&](int buffer) {
    const char* cur = lds + buffer * BUF;
#pragma unroll
    for (int q = 0; q < KT / 16; ++q) {
      shortx8 b[NB][P];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int p = 0; p < P; ++p) b[n][p] = OpB::fragment(cur + OpA::BYTES, p, wj + n * 32, q);
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        shortx8 f[P];
#pragma unroll
        for (int p = 0; p < P; ++p) f[p] = OpA::fragment(cur, p, wi + m * 32, q);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          acc[m][n] = mfma<bf16_t>(f[2], b[n][0], acc[m][n]);
          acc[m][n] = mfma<bf16_t>(f[0], b[n][2], acc[m][n]);
          acc[m][n] = mfma<bf16_t>(f[1], b[n][1], acc[m][n]);
          acc[m][n] = mfma<bf16_t>(f[1], b[n][0], acc[m][n]);
          acc[m][n] = mfma<bf16_t>(f[0], b[n][1], acc[m][n]);
          acc[m][n] = mfma<bf16_t>(f[0], b[n][0], acc[m][n]);
        }
      }
    }
  };
  const int whole = A.inside() && B.inside() ? have / KT : 0;   // stages that need no ends to be cut
  const bool a_edge = A_ACROSS && A.left < BM, b_edge = B_ACROSS && B.left < BN;
  auto fetch = [&](int slot, int stage) {
    if (stage < whole) {
      A.template fetch<true>(slot, KT);
      B.template fetch<true>(slot, KT);
    } else if (stage < stages) {
      A.template fetch<false>(slot, have - stage * KT);
      B.template fetch<false>(slot, have - stage * KT);
    }
  };
  // stage s is multiplied from one buffer while s + 1 goes from its registers into the other and s + 1 + DEPTH is fetched
  auto step = [&](int s, int u, auto only_whole) {
    constexpr bool WHOLE = decltype(only_whole)::value;
    __syncthreads();   // stage s is in LDS for everyone, stage s - 1 has been read by everyone
    const int buffer = DEPTH == 2 ? u : s & 1, slot = (u + 1) % DEPTH;
    multiply(buffer);
    if (WHOLE || s + 1 < stages) {
      const bool w = WHOLE || s + 1 < whole;
      A.store(lds + (1 - buffer) * BUF, slot, w && a_edge, lost);
      B.store(lds + (1 - buffer) * BUF + OpA::BYTES, slot, w && b_edge, lost);
    }
    if (WHOLE) {
      A.template fetch<true>(slot, KT);
      B.template fetch<true>(slot, KT);
    } else {
      fetch(slot, s + 1 + DEPTH);
    }
    if (WHOLE) {
      // the cutting of stage s + 1 runs between the matrix instructions of stage s, up to four of its instructions behind each
      // (16384 x 512 x 512: 53.7 us, one 54.6, six 55)
#pragma unroll
      for (int i = 0; i < MB * NB * 6; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, 4, 0);
      }
    }
  };
  fetch(0, 0);
  A.store(lds, 0, whole > 0 && a_edge, lost);
  B.store(lds + OpA::BYTES, 0, whole > 0 && b_edge, lost);
#pragma unroll
  for (int d = 1; d <= DEPTH; ++d) fetch(d % DEPTH, d);
  int s = 0;
  for (; s + 2 * DEPTH < whole; s += DEPTH)
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) step(s + u, u, std::true_type());
  for (; s < stages; s += DEPTH)
#pragma unroll
    for (int u = 0; u < DEPTH; ++u)
      if (s + u < stages) step(s + u, u, std::false_type());

  static_assert(32 * tile_stride(NB) * 4 * WM * WN <= 2 * BUF, "the turned tiles fit into the stage buffers");
  {
    bool bad = false;
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 16; ++g) bad |= !(fabsf(acc[m][n][g]) <= 3.4028235e38f);
    bool again = __syncthreads_or(bad || (lost & 0xffff));
    if (again && !__syncthreads_or(bad)) {
      // Bits were lost, at most 2^-134 of a value.  Does a sum notice: can all of its products together have lost enough to reach
      // the result's smallest step, and is it below 2^25 times that?  A sum of 0 is one where its row of A or its column of B holds
      // nothing else; lines outside the matrix count as such.
      uint8_t *live_a = (uint8_t*)lds + 64, *live_b = live_a + BM;
      for (int t = threadIdx.x; t < BM + BN; t += THREADS) live_a[t] = 0;
      __syncthreads();
      const float reach = (float)have * (panel_max<A_ACROSS, BM, THREADS>((const float*)a.A, a.lda, i0, min(a.M - i0, BM), k0, have, (float*)lds, live_a) +
                                         panel_max<B_ACROSS, BN, THREADS>((const float*)a.B, a.ldb, j0, min(a.N - j0, BN), k0, have, (float*)lds, live_b));
      if (reach > 0x1p-26f) {   // each part of a split sum (1024 at most) may lose 2^-160, half a step of 2^-149 in all
        const float least = reach * 0x1p-109f;
        const int lane = threadIdx.x & 63;
        bool column[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) column[n] = live_b[wj + n * 32 + (lane & 31)];
#pragma unroll
        for (int m = 0; m < MB; ++m)
#pragma unroll
          for (int g = 0; g < 16; ++g) {
            const bool row = live_a[wi + m * 32 + 4 * (lane >> 5) + (g & 3) + 8 * (g >> 2)];
#pragma unroll
            for (int n = 0; n < NB; ++n) bad |= fabsf(acc[m][n][g]) < least && (acc[m][n][g] != 0.0f || (row && column[n]));
          }
      }
      again = __syncthreads_or(bad);
    }
    if (again) fp32_sums<A_ACROSS, B_ACROSS, MB, NB>(a, i0 + wi, j0 + wj, k0, have, acc);
  }
  tile_end<float, MB, NB, WM * WN>(a, split, i0 + wi, j0 + wj, acc, (float*)lds);
}

template <bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN, int DEPTH>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_tile32(TileArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  tile32<A_ACROSS, B_ACROSS, BM, BN, WM, WN, DEPTH>(a, blockIdx.x, lds);
}

// ---- k_tile16 ------------------------------------------------------------------------------------------------------
// bf16 and fp16.  A ring of LDS stages of 32 r is filled by DMA (global_load_lds_dwordx4: no registers, no LDS store
// instructions), so all but one of its stages are on their way while one is multiplied.  Two steps of 16 r a stage, and
// the fragments of a step are read while the step before is multiplied; the one barrier of a stage lies between its two
// steps, when the second step's fragments are in registers: no wave waits for LDS behind it.  Bound by the matrix cores, then
// by the epilogue, which no other workgroup of the CU covers: 65536 x 1536 x 512 bf16 91 us (1.13 PFLOP/s), its weight's
// gradient 86 and the input's, with three times the results, 117; 4096^3 110 to 125 (a library product 91 to 125).
//
// A wave's DMA writes 1 KB of LDS in lane order, from any 16-byte pieces of memory.  Along r, LDS holds [i][32 r] (64
// bytes), and the four pieces of a row are exchanged by (i >> 2) & 3: sixteen lanes of a fragment, sixteen rows, touch
// all 64 banks.  Across r it holds [r][i], pieces exchanged by (r & 3) << 2: the four rows that 32 lanes read through
// ds_read_b64_tr_b16, 64 bytes of each, lie on different banks.  Needs operands on 16-byte boundaries; others are copied
// first (k_pack).  In the last stage, where r is not a multiple of 32, every lane clears what it has fetched behind the end.
constexpr int KT16 = 32;
template <typename T, bool ACROSS, int ROWS, int WAVES, int BLOCKS>
struct Operand16 {
  static constexpr int BYTES = ROWS * KT16 * 2, PIECES = BYTES / 1024 / WAVES, PER_LINE = (ACROSS ? ROWS : KT16) / 8;
  static_assert(PIECES * 1024 * WAVES == BYTES, "pieces");
  const char* base;        // uniform: the stage to come
  int64_t step;            // bytes between stages
  unsigned off[PIECES];    // this lane's piece, relative to base
  unsigned line_bytes;

  __device__ __forceinline__ static int line_of(int p) { return ((threadIdx.x >> 6) * PIECES + p) * (64 / PER_LINE) + (threadIdx.x & 63) / PER_LINE; }
  __device__ __forceinline__ static int piece_of(int line) {
    return ((threadIdx.x & 63) % PER_LINE) ^ (ACROSS ? (line & 3) << 2 : (line >> 2) & 3);
  }
  __device__ __forceinline__ void init(const void* p, int64_t ld, int i0, int n_i, int64_t k0) {
    const int left = n_i - i0;
    line_bytes = (unsigned)ld * 2;
    base = (const char*)p + (ACROSS ? k0 * ld + i0 : (int64_t)i0 * ld + k0) * 2;
    step = (ACROSS ? KT16 * ld : KT16) * 2;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int line = line_of(p), c = piece_of(line) * 8;
      // outside the matrix: its last row, its first columns; they only reach sums nobody stores
      off[p] = ACROSS ? (unsigned)(line * ld + (c < left ? c : 0)) * 2 : (unsigned)((line < left ? line : left - 1) * ld + c) * 2;
    }
  }
  // the next stage into LDS at dst; have: r values that exist from it on.  Pieces wholly behind the end come from the
  // stage's first one; a piece that holds the end is read whole (16 aligned bytes never leave the memory of their first)
  __device__ __forceinline__ void fetch(char* dst, int have) {
    const unsigned m0 = (unsigned)(size_t)(lds_char*)dst + (threadIdx.x >> 6) * (PIECES * 1024);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int line = line_of(p);
      const bool in = have >= KT16 || (ACROSS ? line : piece_of(line) * 8) < have;
      const unsigned o = in ? off[p] : off[p] - (ACROSS ? line * line_bytes : (unsigned)piece_of(line) * 16);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(m0 + p * 1024)),
                   "v"(o), "s"(base)
                   : "memory");
    }
    base += step;
  }
  // piece p of the next stage, all of whose r values exist; after the last one, advance().  M0 holds a DMA's LDS address;
  // hipcc has no use of its own for it here (LDS instructions of gfx9 do not read it).
  __device__ __forceinline__ void fetch_piece(char* dst, int p) const {
    const unsigned m0 = (unsigned)(size_t)(lds_char*)dst + (threadIdx.x >> 6) * (PIECES * 1024) + p * 1024;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(m0)), "v"(off[p]), "s"(base)
                 : "memory");
  }
  __device__ __forceinline__ void advance() { base += step; }
  // clears this lane's values behind the end of a landed stage
  __device__ __forceinline__ static void clear(char* dst, int have) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int line = line_of(p), n = ACROSS ? (line < have ? 8 : 0) : have - piece_of(line) * 8;
      if (n >= 8) continue;
      T* at = (T*)(dst + ((threadIdx.x >> 6) * PIECES + p) * 1024 + (threadIdx.x & 63) * 16);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= n) at[i] = (T)0.0f;
    }
  }
  // byte offsets of this lane's part of a wave's fragments, whose i values start at iw (a multiple of 32): along r one for
  // each step of 16 r, across r one for each block of 32 i
  static constexpr int OFFSETS = ACROSS ? BLOCKS : 2;
  __device__ __forceinline__ static void lane_offsets(int iw, unsigned (&o)[OFFSETS]) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int v = 0; v < OFFSETS; ++v) {
      if (ACROSS) {
        const int q = lane & 15, r = q >> 2;
        const int piece = ((iw / 8 + v * 4) | ((lane & 16) >> 3) | ((q & 3) >> 1)) ^ (r << 2);
        o[v] = (8 * h + r) * (ROWS * 2) + piece * 16 + (q & 1) * 8;
      } else {
        const int r = lane & 31;
        o[v] = (iw + r) * 64 + (((2 * v + h) ^ ((r >> 2) & 3)) * 16);
      }
    }
  }
  // fragment of 32 i values of block `block`, 16 r values from 16 s
  __device__ __forceinline__ static shortx8 fragment(const char* lds, const unsigned (&o)[OFFSETS], int block, int s) {
    if constexpr (ACROSS) {
      const char* p = lds + o[block] + s * (16 * ROWS * 2);
      const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(p));
      const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(p + 4 * ROWS * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *(const shortx8*)(lds + o[s] + block * (32 * 64));
    }
  }
};

template <typename T, bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN, int RING>
__device__ __forceinline__ void tile16(const TileArgs& a, int block, char* lds) {
  constexpr int WAVES = WM * WN, MB = BM / WM / 32, NB = BN / WN / 32;
  typedef Operand16<T, A_ACROSS, BM, WAVES, MB> OpA;
  typedef Operand16<T, B_ACROSS, BN, WAVES, NB> OpB;
  constexpr int BUF = OpA::BYTES + OpB::BYTES, LOADS = OpA::PIECES + OpB::PIECES;
  static_assert(32 * tile_stride(NB) * 4 * WAVES <= RING * BUF, "the turned tiles fit into the ring");
  static_assert(RING == 3 || RING == 4, "waits");
  static_assert(MB * NB >= MB + NB && MB * NB >= LOADS, "one fragment and one load a matrix instruction");
  const TilePlace at = tile_place(a, block, BM, BN);
  const int64_t k0 = at.split * a.per;
  const int have = (int)(a.K - k0 < a.per ? a.K - k0 : a.per), whole = have / KT16, rest = have % KT16, stages = whole + (rest ? 1 : 0);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = wave / WN * (MB * 32), wj = wave % WN * (NB * 32);

  floatx16 acc[MB][NB];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int g = 0; g < 16; ++g) acc[m][n][g] = 0.0f;
  OpA A;
  OpB B;
  A.init(a.A, a.lda, at.i0, a.M, k0);
  B.init(a.B, a.ldb, at.j0, a.N, k0);
  unsigned oa[OpA::OFFSETS], ob[OpB::OFFSETS];
  OpA::lane_offsets(wi, oa);
  OpB::lane_offsets(wj, ob);
  auto slot = [&](int t) { return lds + (RING == 4 ? t & 3 : t % 3) * BUF; };
  auto fetch = [&](int t) {
    if (t >= stages) return;
    A.fetch(slot(t), have - t * KT16);
    B.fetch(slot(t) + OpA::BYTES, have - t * KT16);
  };
  shortx8 fa[2][MB], fb[2][NB];
  auto read = [&](int t, int s) {
    const char* p = slot(t);
#pragma unroll
    for (int n = 0; n < NB; ++n) fb[s][n] = OpB::fragment(p + OpA::BYTES, ob, n, s);
#pragma unroll
    for (int m = 0; m < MB; ++m) fa[s][m] = OpA::fragment(p, oa, m, s);
  };
  auto multiply = [&](int s) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[m][n] = mfma<T>(fa[s][m], fb[s][n], acc[m][n]);
  };
  // stage t has landed for everyone, and everyone has read what it wants of the stage before.  Stages up to
  // t + RING - 2 are under way, LOADS loads of this wave each.
  auto meet = [&](int t) {
    const int behind = min(t + RING - 1, stages) - (t + 1);
    if (RING == 4 && behind >= 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * LOADS) : "memory");
    else if (behind >= 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
#pragma unroll 1
  for (int t = 0; t < RING - 1; ++t) fetch(t);
  if (whole) {
    meet(0);
    fetch(RING - 1);
    read(0, 0);
    int t = 0;
    // Where the stage to fetch exists and is whole: fragments and DMA are issued one after each matrix instruction, so that
    // neither delays the next one (all of them behind the barrier left the matrix cores idle for a fifth of a stage).
    for (; t + RING < whole; ++t) {
      const char *cur = slot(t), *next = slot(t + 1);
      char* dst = slot(t);
#pragma unroll
      for (int i = 0; i < MB * NB; ++i) {
        acc[i / NB][i % NB] = mfma<T>(fa[0][i / NB], fb[0][i % NB], acc[i / NB][i % NB]);
        if (i < NB) fb[1][i] = OpB::fragment(cur + OpA::BYTES, ob, i, 1);
        else if (i < NB + MB) fa[1][i - NB] = OpA::fragment(cur, oa, i - NB, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((RING - 2) * LOADS) : "memory");
#pragma unroll
      for (int i = 0; i < MB * NB; ++i) {
        acc[i / NB][i % NB] = mfma<T>(fa[1][i / NB], fb[1][i % NB], acc[i / NB][i % NB]);
        if (i < NB) fb[0][i] = OpB::fragment(next + OpA::BYTES, ob, i, 0);
        else if (i < NB + MB) fa[0][i - NB] = OpA::fragment(next, oa, i - NB, 0);
        if (i < OpA::PIECES) A.fetch_piece(dst, i);
        else if (i < LOADS) B.fetch_piece(dst + OpA::BYTES, i - OpA::PIECES);
        __builtin_amdgcn_sched_barrier(0);
      }
      A.advance();
      B.advance();
    }
    for (; t < whole; ++t) {
      read(t, 1);
      multiply(0);
      if (t + 1 < whole) {
        meet(t + 1);
        fetch(t + RING);
        read(t + 1, 0);
      }
      multiply(1);
    }
  }
  if (rest) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    OpA::clear(slot(whole), rest);
    OpB::clear(slot(whole) + OpA::BYTES, rest);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    read(whole, 0);
    multiply(0);
    read(whole, 1);
    multiply(1);
  }
  tile_end<T, MB, NB, WAVES>(a, at.split, at.i0 + wi, at.j0 + wj, acc, (float*)lds);
}

template <typename T, bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN, int RING>
__global__ __launch_bounds__(WM * WN * 64, RING == 3 ? 3 : 2) void k_tile16(TileArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  tile16<T, A_ACROSS, B_ACROSS, BM, BN, WM, WN, RING>(a, blockIdx.x, lds);
}

// Both gradients of a layer in one launch where neither fills the chip: the first `split` workgroups compute dx, the others dW
// (4099 rows of 515 x 257 in fp32, 165 and 255 workgroups: 36 us, 50 one after the other).
template <typename T, bool W_NK>
__global__ __launch_bounds__(256, 2) void k_tile_pair(TileArgs dx, TileArgs dw, int split) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int block = blockIdx.x;
  if constexpr (sizeof(T) == 4) {
    if (block < split) tile32<false, W_NK, 128, 128, 2, 2, 2>(dx, block, lds);
    else tile32<true, true, 128, 128, 2, 2, 2>(dw, block - split, lds);
  } else {
    if (block < split) tile16<T, false, W_NK, 128, 128, 2, 2, 4>(dx, block, lds);
    else tile16<T, true, true, 128, 128, 2, 2, 4>(dw, block - split, lds);
  }
}

// a copy of a 16-bit matrix on 16-byte boundaries
template <typename T>
__global__ __launch_bounds__(256) void k_pack(const T* __restrict__ src, int64_t lds_, T* __restrict__ dst, int64_t ldd, int64_t rows, int cols) {
  const int64_t per = ldd / 8, total = rows * per;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / per;
    const int c = (int)(t - r * per) * 8;
    const Vec<T> v = load_vec(src + r * lds_ + c, cols - c, c);
    store_vec(dst + r * ldd + c, v, 8);
  }
}

// ---- k_small -------------------------------------------------------------------------------------------------------
// Small products are bound by latency, not by the matrix cores: operands go straight from memory (or L2) into fragments
// of v_mfma_f32_16x16x4, 16-bit types widened (exact), 16 r values a step.  Eight waves a workgroup: long sums
// (KS = 8) give every wave an eighth of the steps of one 16 x 16 tile and add the eight in order; short ones (KS = 1) give
// every wave a tile of its own.  An operand can be gated, dz = dy act'(pre), as it is read, and its sum over r
// (the bias's gradient) taken along: a backward pass of this size is one launch.  24 x 1024 x 512 fp32 forward 5.6 us, both
// gradients of 32 x 1024 x 512 7.4 us: a launch of nothing is 2.5.
struct SmallOperand {
  const void* p;
  const void* gate;   // z, or null
  int64_t ld, ldg;
};
struct SmallArgs {
  SmallOperand A, B;
  int M, N, K, mt, nt, ks, act;
  void* rsum;         // sum over r of operand B (rsum_of_a: of A), or null
  int rsum_of_a;
  Epilogue e;
};
constexpr int SMALL_WAVES = 8;

template <typename T, bool ACROSS, bool GATED, bool FULL>
__device__ __forceinline__ floatx4 small_operand(const SmallOperand& o, int i, int r0, int K, int act) {
  floatx4 v = load_4r<T, ACROSS, FULL>(o.p, o.ld, i, r0, K);
  if constexpr (GATED) {
    if (act != DISN_ACT_NONE) {
      const floatx4 z = load_4r<T, ACROSS, FULL>(o.gate, o.ldg, i, r0, K);
      float g[4] = {v[0], v[1], v[2], v[3]};
      gate_all<T>(g, z, act);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = FULL || r0 + e < K ? g[e] : 0.0f;
    }
  }
  return v;
}

template <typename T, bool A_ACROSS, bool B_ACROSS, bool A_GATED, bool B_GATED, int KS>
__device__ __forceinline__ void small_product(const SmallArgs& a, int block, float (*lds)[256], float (*lds_sum)[16]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), idx = lane & 15, quad = lane >> 4;
  constexpr int JW = SMALL_WAVES / KS;   // tiles along j of a workgroup
  const int nt = (a.nt + JW - 1) / JW, ti = block / nt, tj = (block - ti * nt) * JW + (KS == 1 ? wave : 0);
  const int i0 = ti * 16, j0 = tj * 16;
  if (KS == 1 && tj >= a.nt) return;
  const int i = min(i0 + idx, a.M - 1), j = min(j0 + idx, a.N - 1);
  const int full = a.K >> 4;
  floatx4 acc = {0, 0, 0, 0};
  float sum = 0.0f;
  auto step = [&](floatx4 av, floatx4 bv) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(av[e], bv[e], acc, 0, 0, 0);
    if constexpr (A_GATED || B_GATED) {
      const floatx4 g = a.rsum_of_a ? av : bv;
      sum += (g[0] + g[1]) + (g[2] + g[3]);
    }
  };
  int c = KS == 1 ? 0 : wave;
  for (; c + 3 * KS < full; c += 4 * KS) {
    floatx4 av[4], bv[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      av[u] = small_operand<T, A_ACROSS, A_GATED, true>(a.A, i, (c + u * KS) * 16 + quad * 4, a.K, a.act);
      bv[u] = small_operand<T, B_ACROSS, B_GATED, true>(a.B, j, (c + u * KS) * 16 + quad * 4, a.K, a.act);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) step(av[u], bv[u]);
  }
  for (; c < full; c += KS)
    step(small_operand<T, A_ACROSS, A_GATED, true>(a.A, i, c * 16 + quad * 4, a.K, a.act),
         small_operand<T, B_ACROSS, B_GATED, true>(a.B, j, c * 16 + quad * 4, a.K, a.act));
  if ((a.K & 15) && c == full)
    step(small_operand<T, A_ACROSS, A_GATED, false>(a.A, i, c * 16 + quad * 4, a.K, a.act),
         small_operand<T, B_ACROSS, B_GATED, false>(a.B, j, c * 16 + quad * 4, a.K, a.act));
  const bool want_sum = (A_GATED || B_GATED) && a.rsum && (a.rsum_of_a ? tj == 0 : ti == 0);
  if (A_GATED || B_GATED) {
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
  }
  // lane's place in the tile: j = l & 15, i = 4 (l >> 4) + g
  if constexpr (KS == 1) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (i0 + quad * 4 + g < a.M && j0 + idx < a.N) finish_one<T>(a.e, i0 + quad * 4 + g, j0 + idx, acc[g]);
    const int at = (a.rsum_of_a ? i0 : j0) + idx;
    if (want_sum && quad == 0 && at < (a.rsum_of_a ? a.M : a.N)) ((T*)a.rsum)[at] = (T)sum;
  } else {
#pragma unroll
    for (int g = 0; g < 4; ++g) lds[wave][(quad * 4 + g) * 16 + idx] = acc[g];
    if (quad == 0) lds_sum[wave][idx] = sum;
    __syncthreads();
    const int t = threadIdx.x;
    if (t < 256) {
      float z = lds[0][t];
#pragma unroll
      for (int w = 1; w < KS; ++w) z += lds[w][t];
      if (i0 + (t >> 4) < a.M && j0 + (t & 15) < a.N) finish_one<T>(a.e, i0 + (t >> 4), j0 + (t & 15), z);
    } else if (want_sum && t < 272) {
      float z = lds_sum[0][t & 15];
#pragma unroll
      for (int w = 1; w < KS; ++w) z += lds_sum[w][t & 15];
      const int at = (a.rsum_of_a ? i0 : j0) + (t & 15);
      if (at < (a.rsum_of_a ? a.M : a.N)) ((T*)a.rsum)[at] = (T)z;
    }
  }
}

template <typename T, bool B_ACROSS>
__global__ __launch_bounds__(SMALL_WAVES * 64) void k_small(SmallArgs a) {
  __shared__ float lds[SMALL_WAVES][256];
  __shared__ float lds_sum[SMALL_WAVES][16];
  if (a.ks == 1) small_product<T, false, B_ACROSS, false, false, 1>(a, blockIdx.x, lds, lds_sum);
  else small_product<T, false, B_ACROSS, false, false, SMALL_WAVES>(a, blockIdx.x, lds, lds_sum);
}
// dx and dW (with the bias's gradient) of one layer in one launch: the first `split` workgroups compute dx
template <typename T, bool W_NK>
__global__ __launch_bounds__(SMALL_WAVES * 64) void k_small_backward(SmallArgs dx, SmallArgs dw, int split) {
  __shared__ float lds[SMALL_WAVES][256];
  __shared__ float lds_sum[SMALL_WAVES][16];
  if ((int)blockIdx.x < split) {
    if (dx.ks == 1) small_product<T, false, W_NK, true, false, 1>(dx, blockIdx.x, lds, lds_sum);
    else small_product<T, false, W_NK, true, false, SMALL_WAVES>(dx, blockIdx.x, lds, lds_sum);
  } else {
    if (dw.ks == 1) small_product<T, true, true, W_NK, !W_NK, 1>(dw, blockIdx.x - split, lds, lds_sum);
    else small_product<T, true, true, W_NK, !W_NK, SMALL_WAVES>(dw, blockIdx.x - split, lds, lds_sum);
  }
}

// ---- k_rows: few rows times a large matrix ---------------------------------------------------------------------------
// W is read once at memory speed, each value multiplied with MR rows of x by fp32 FMAs.  W by rows of r (across): a lane owns 16 bytes of columns, the workgroup's
// four waves share a range of r, ranges become partial sums for k_finish.  1 x 4096 x 4096 fp32: 12.5 us (5.4 TB/s) and 4 us of
// k_finish.
struct RowsArgs {
  const void *x, *w;
  int64_t ldx, ldw;
  int M, N, K, per, groups;   // per: r values of a workgroup; groups: workgroups along the columns
  float* part;
  Epilogue e;
};
constexpr int ROWS_MAX_PER = 128;

template <typename T, int MR>
__global__ __launch_bounds__(256) void k_rows_across(RowsArgs a) {
  constexpr int V = Vec<T>::N;
  __shared__ float xs[ROWS_MAX_PER * MR];
  __shared__ float red[4][64 * V];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int group = blockIdx.x % a.groups, split = blockIdx.x / a.groups;
  const int k0 = split * a.per, have = min(a.per, a.K - k0);
  for (int t = threadIdx.x; t < have * MR; t += 256) {
    const int m = t / have, k = t - m * have;
    xs[k * MR + m] = m < a.M ? (float)((const T*)a.x)[m * a.ldx + k0 + k] : 0.0f;
  }
  __syncthreads();
  const int col = (group * 64 + lane) * V, n = a.N - col;
  const T* w = (const T*)a.w + (int64_t)k0 * a.ldw + (n > 0 ? col : 0);
  float acc[MR][V];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int i = 0; i < V; ++i) acc[m][i] = 0.0f;
  auto add = [&](int k, const Vec<T>& v) {
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const float x = xs[k * MR + m];
#pragma unroll
      for (int i = 0; i < V; ++i) acc[m][i] = fmaf(x, (float)v.v[i], acc[m][i]);
    }
  };
  if (n >= V || n <= 0) {   // lanes behind the last column read the first ones; their sums are not stored
    const bool wide = a.N >= V;
    int k = wave;
    for (; wide && k + 28 < have; k += 32) {
      Vec<T> v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = load_vec(w + (int64_t)(k + 4 * u) * a.ldw);
#pragma unroll
      for (int u = 0; u < 8; ++u) add(k + 4 * u, v[u]);
    }
    for (; k < have; k += 4) add(k, load_vec(w + (int64_t)k * a.ldw, wide ? V : a.N, 0));
  } else {
    for (int k = wave; k < have; k += 4) add(k, load_vec(w + (int64_t)k * a.ldw, n, col));
  }
#pragma unroll
  for (int m = 0; m < MR; ++m) {
    if (m > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) red[wave][lane * V + i] = acc[m][i];
    __syncthreads();
    for (int t = threadIdx.x; t < 64 * V; t += 256) {
      const int j = group * 64 * V + t;
      if (m < a.M && j < a.N) a.part[((size_t)split * a.M + m) * a.N + j] = (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
    }
  }
}

// W by rows of j (along r): a workgroup owns NR rows of W, its lanes run along r.
template <typename T, int MR, int NR>
__global__ __launch_bounds__(256) void k_rows_along(RowsArgs a) {
  constexpr int V = Vec<T>::N;
  __shared__ float red[4][MR * NR];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j0 = blockIdx.x * NR;
  const T* w[NR];
#pragma unroll
  for (int j = 0; j < NR; ++j) w[j] = (const T*)a.w + (int64_t)min(j0 + j, a.N - 1) * a.ldw;
  float acc[MR][NR];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < NR; ++j) acc[m][j] = 0.0f;
  for (int k = threadIdx.x * V; k < a.K; k += 256 * V) {
    const int n = a.K - k;
    Vec<T> wv[NR];
#pragma unroll
    for (int j = 0; j < NR; ++j) wv[j] = load_vec(w[j] + k, n, k);
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      const Vec<T> xv = load_vec((const T*)a.x + min(m, a.M - 1) * a.ldx + k, n, k);
#pragma unroll
      for (int j = 0; j < NR; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[m][j] = fmaf((float)xv.v[i], (float)wv[j].v[i], acc[m][j]);
    }
  }
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      float s = acc[m][j];
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
      if (lane == 0) red[wave][m * NR + j] = s;
    }
  __syncthreads();
  if (threadIdx.x < MR * NR) {
    const int m = threadIdx.x / NR, j = j0 + threadIdx.x % NR;
    if (m < a.M && j < a.N)
      finish_one<T>(a.e, m, j, (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]));
  }
}

// ---- k_outer: sums of up to 8 products ---------------------------------------------------------------------------------
// (the first layer of three coordinates; gradients of a layer with few outputs or of few rows).  Bound by writing C: a lane
// keeps its 16 bytes of columns of B and walks over rows, several of them under way.
// 262144 x 512 results of one product: bf16 54 us (5.0 TB/s), k_small 152; fp32 109 and 186; of three products in fp32, 65536
// rows 36 and 45.  In 16 bits more products are faster in tiles (65536 x 512 of three 24 us, here 37; but 262144 x 64 here 25,
// k_small 35).
struct OuterArgs {
  const void *A, *B;
  int64_t ai, ar, bj, br;   // distances along i, j and r
  int64_t M, rows_per;
  int N, K, lanes, groups;
  Epilogue e;
};
constexpr int THIN = 8;     // the longest sum of k_outer, the widest narrow operand of k_thin
template <typename T, int KR>
__global__ __launch_bounds__(256) void k_outer(OuterArgs a) {
  constexpr int V = Vec<T>::N, U = 4;
  const int L = a.lanes, sub = threadIdx.x % L, line = threadIdx.x / L, lines = 256 / L;
  const int group = blockIdx.x % a.groups;
  const int64_t i0 = (int64_t)(blockIdx.x / a.groups) * a.rows_per, i1 = min(a.M, i0 + a.rows_per);
  const int col = (group * L + sub) * V, n = a.N - col;
  if (n <= 0) return;
  float b[KR][V];
#pragma unroll
  for (int k = 0; k < KR; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) b[k][v] = k < a.K && v < n ? (float)((const T*)a.B)[(col + v) * a.bj + k * a.br] : 0.0f;
  const Vec<T> bias = bias_vec<T>(a.e, col, n);
  for (int64_t i = i0 + line; i < i1; i += U * lines) {
    float x[U][KR];
    Vec<T> res[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = min(i + u * lines, i1 - 1);
#pragma unroll
      for (int k = 0; k < KR; ++k) x[u][k] = k < a.K ? (float)((const T*)a.A)[row * a.ai + k * a.ar] : 0.0f;
      res[u] = residual_vec<T>(a.e, row, col, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = i + u * lines;
      if (row >= i1) break;
      float z[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        z[v] = x[u][0] * b[0][v];
#pragma unroll
        for (int k = 1; k < KR; ++k)
          if (k < a.K) z[v] = fmaf(x[u][k], b[k][v], z[v]);
      }
      finish_vec<T>(a.e, (T*)a.e.out + row * a.e.ldo + col, (T*)a.e.pre + row * a.e.ldp + col, z, n, bias, res[u]);
    }
  }
}

// ---- k_thin: long sums of a wide and a narrow operand, both across r -----------------------------------------------------
// (the weight's gradient of a layer with few outputs or few inputs).  Bound by reading the wide operand: a lane owns 16 bytes
// of its columns and sums their products with each of up to 8 columns of the narrow one; parts of r become partial sums.
// Weight's gradient over 262144 rows of 512 inputs and one output, fp32: 104 us (5.2 TB/s), 356 in tiles.  fp32 only: in 16
// bits the tiles are as fast (65536 x 512, one output: 20 us both).
struct ThinArgs {
  const float *wide, *narrow;
  int64_t ldw, ldn, K, rows_per;
  int D, S, lanes, groups;
  int64_t od, os, size;   // places in C of the wide operand's columns, the narrow one's, and of all
  float* part;
};
template <int SR>
__global__ __launch_bounds__(256) void k_thin(ThinArgs a) {
  constexpr int V = 4, U = 8;
  __shared__ float red[4][64 * V];
  const int L = a.lanes, sub = threadIdx.x % L, line = threadIdx.x / L, lines = 256 / L, wave = threadIdx.x >> 6;
  const int group = blockIdx.x % a.groups;
  const int64_t split = blockIdx.x / a.groups, r0 = split * a.rows_per, r1 = min(a.K, r0 + a.rows_per);
  const int col = (group * L + sub) * V, back = col < a.D && col + V > a.D ? col + V - a.D : 0;
  const float* w = a.wide + (col < a.D ? col - back : 0);   // lanes behind the last column: the first ones, not stored
  const bool ragged = (group + 1) * L * V > a.D;
  float acc[SR][V];
#pragma unroll
  for (int s = 0; s < SR; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) acc[s][v] = 0.0f;
  for (int64_t r = r0 + line; r < r1; r += U * lines) {
    Vec<float> x[U];
    float t[U][SR];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = min(r + u * lines, r1 - 1);
      x[u] = load_vec(w + row * a.ldw);
#pragma unroll
      for (int s = 0; s < SR; ++s) t[u][s] = s < a.S ? a.narrow[row * a.ldn + s] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r + u * lines >= r1) break;
      if (ragged) x[u] = shift_vec(x[u], back);
#pragma unroll
      for (int s = 0; s < SR; ++s)
        if (s < a.S) {
#pragma unroll
          for (int v = 0; v < V; ++v) acc[s][v] = fmaf(x[u].v[v], t[u][s], acc[s][v]);
        }
    }
  }
#pragma unroll
  for (int s = 0; s < SR; ++s) {
    if (s >= a.S) break;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      for (int d = L; d < 64; d <<= 1) acc[s][v] += __shfl_xor(acc[s][v], d, 64);
      if ((threadIdx.x & 63) < L) red[wave][sub * V + v] = acc[s][v];
    }
    __syncthreads();
    for (int t = threadIdx.x; t < L * V; t += 256) {
      const int j = group * L * V + t;
      if (j < a.D) a.part[split * a.size + j * a.od + s * a.os] = (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
    }
    __syncthreads();
  }
}

// ---- dz = dy act'(pre) and partial column sums of it -------------------------------------------------------------------
// A lane owns 16 bytes of columns (SINGLE: one, for rows of less than 16 bytes); rows narrower than a wave put several of them
// into it.  Four rows are under way.  Bound by memory: 65536 x 512 bf16 relu 38 us, 5.3 TB/s
// of the three matrices.
struct GateArgs {
  const void *dy, *pre;
  void* dz;          // null: only the sums
  float* part;       // [row blocks][N] or null
  int64_t lddy, ldp, ldz, M, rows_per;
  int N, lanes, groups, act;
};
template <typename T, bool SINGLE>
__global__ __launch_bounds__(256) void k_gate(GateArgs a) {
  constexpr int V = SINGLE ? 1 : Vec<T>::N, U = 4;
  __shared__ float red[4][64 * V];
  const int L = a.lanes, sub = threadIdx.x % L, line = threadIdx.x / L, lines = 256 / L;
  const int group = blockIdx.x % a.groups;
  const int64_t rb = blockIdx.x / a.groups;
  const int col = (group * L + sub) * V, n = a.N - col, back = !SINGLE && n > 0 && n < V ? V - n : 0;
  const int at = n > 0 ? col - back : 0;   // where a lane reads: the last piece further in front, and shifted
  const int64_t r1 = min(a.M, (rb + 1) * a.rows_per);
  const bool ragged = !SINGLE && (group + 1) * L * V > a.N;
  auto load = [&](const void* p, int64_t ld, int64_t row, Vec<T>& v) {
    if constexpr (SINGLE) v.v[0] = ((const T*)p)[row * ld + at];
    else v = load_vec((const T*)p + row * ld + at);
  };
  float s[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.0f;
  for (int64_t r = rb * a.rows_per + line; r < r1; r += U * lines) {
    Vec<T> g[U], z[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = min(r + u * lines, r1 - 1);
      load(a.dy, a.lddy, row, g[u]);
      if (a.act != DISN_ACT_NONE) load(a.pre, a.ldp, row, z[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = r + u * lines;
      if (row >= r1) break;
      if (ragged) {
        g[u] = shift_vec(g[u], back);
        if (a.act != DISN_ACT_NONE) z[u] = shift_vec(z[u], back);
      }
      float v[V];
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = (float)g[u].v[i];
      if (a.act != DISN_ACT_NONE) gate_all<T>(v, z[u].v, a.act);
      if (a.dz && n > 0) {
        T* dz = (T*)a.dz + row * a.ldz + col;
        if constexpr (SINGLE) {
          *dz = (T)v[0];
        } else {
          Vec<T> o;
          narrow<T, V>(v, o.v);
          store_vec(dz, o, n);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += v[i];
    }
  }
  if (!a.part) return;
  // a wave's rows by lane exchange, the four waves through LDS
#pragma unroll
  for (int i = 0; i < V; ++i) {
    for (int d = L; d < 64; d <<= 1) s[i] += __shfl_xor(s[i], d, 64);
    if ((threadIdx.x & 63) < L) red[threadIdx.x >> 6][sub * V + i] = s[i];
  }
  __syncthreads();
  for (int t = threadIdx.x; t < L * V; t += 256) {
    const int j = group * L * V + t;
    if (j < a.N) a.part[(size_t)rb * a.N + j] = (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
  }
}

// ---- host: which kernel, which tile ------------------------------------------------------------------------------------
enum Kind { K_EMPTY, K_SMALL, K_ROWS, K_OUTER, K_THIN, K_TILE };
struct Product {
  const void *A, *B;
  int64_t lda, ldb;
  bool a_across, b_across;
  int64_t M, N, K;
  Epilogue e;
};
struct Plan {
  Kind kind;
  double us;                 // estimate
  int tile;                  // 128 or 256
  int splits;
  int64_t per;
  int64_t cut;               // > 0: only these rows, in whole rounds of tiles; the others by a plan of their own
  size_t pack_a, pack_b;     // bytes of copies on 16-byte boundaries (k_tile16), 0: none
  size_t bytes;              // of workspace: the copies, then the partial sums
};
size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
// k_tile16 reads 16-byte pieces at 32-bit offsets from a tile's first value
bool tile16_ready(const void* p, int64_t ld) { return dense_aligned(p, 16) && ld % 8 == 0 && ld <= DISN_LINEAR_MAX; }
static_assert(255ll * DISN_LINEAR_MAX * 2 + 64 < 1ll << 32, "offsets of the 256 lines of a tile");
size_t pack_bytes(int64_t rows, int64_t cols) { return align256((size_t)rows * ((cols + 7) / 8 * 8) * 2); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a large product is cut into workgroups: 128- or 256-wide tiles, r split into `splits` parts or not.  A CU holds one
// workgroup with 256-wide tiles (its LDS), two with 128-wide ones, or three of those with a ring of three stages.  A round of
// them costs a fixed time and a time per r value; measured (us, ns per r), 2048 .. 8192 x 1024 .. 4096, r = 512 and 2048:
//              256-wide: half the chip, all of it    128-wide: one a CU    two         three
//   16 bits    9.5, 17                 9.5, 25                 5.5, 7.5     7, 16.5     7.7, 25.5
//   fp32       14, 105                 14, 145                 9.2, 50      9, 85
// Split sums are written and read once more in fp32, at 10 TB/s while they fit the last cache, by one more launch (4 us).
// Measured (estimated): gradient of a 1536 x 512 weight over 65536 bf16 rows 256-wide / 21 parts 107 (105), 128-wide / 10 parts
// 136 (125); 4096 x 4096, r = 2048 256-wide 59 (61), 128-wide 89 (81); 2048 x 2048, r = 2048, 256-wide / 4 parts 39 (40), 128-wide
// 23.  The table's kernels, measured again with results stored past the caches, lie within 10 % of it.  What a tile's end does is not
// priced: 10007 x 777 fp16 results of r = 1000 with a gelu, a residual and z are estimated at 28 and take 50.
// A last round that is at most half full is not started (operands that are copied first aside): the rows before it are one
// launch, the others another (100000 x 512 fp32 outputs are 782 tiles, three rounds and 14 tiles).
struct TileChoice {
  int tile, splits;
  int64_t cut;
  double us;
};
double tile_rounds_us(bool f32, int tile, int64_t blocks, double r) {
  if (tile == 256) {
    const double fill = (double)(blocks % 256) / 256, rounds = (double)(blocks / 256);
    return f32 ? rounds * (14 + 0.145 * r) + (fill > 0 ? 14 + (0.065 + 0.08 * fill) * r : 0)
               : rounds * (9.5 + 0.025 * r) + (fill > 0 ? 9.5 + (0.009 + 0.016 * fill) * r : 0);
  }
  const double one = f32 ? 9.2 + 0.05 * r : 5.5 + 0.0075 * r, two = f32 ? 9 + 0.085 * r : 7 + 0.0165 * r;
  const int64_t full = f32 ? 512 : 768, last = blocks > 512 ? blocks % full : blocks;
  const double three = 7.7 + 0.0255 * r, whole = blocks > 512 ? (double)(blocks / full) * (f32 ? two : three) : 0;
  return whole + (last == 0 ? 0 : last <= 256 ? one : last <= 512 ? two : three);
}
TileChoice choose_tile(bool f32, int64_t M, int64_t N, int64_t K, bool may_cut) {
  TileChoice best{0, 0, 0, 1e30};
  for (int tile = 256; tile >= 128; tile /= 2) {
    const int64_t tiles = ceil_div(M, tile) * ceil_div(N, tile);
    // not split, a few parts, as many as fill the chip in one, two or three workgroups a CU, or as many as the sum allows
    const int64_t parts[] = {1, 2, 3, 4, 128 / tiles, 256 / tiles, 512 / tiles, 768 / tiles, K / 256, K / 128};
    for (const int64_t s : parts) {
      if (s < 1 || (s > 1 && (K / s < 128 || tiles * s > 768))) continue;
      double us = tile_rounds_us(f32, tile, tiles * s, (double)ceil_div(K, s));
      const double moved = 8e-6 * s * M * N;   // MB
      if (s > 1) us += 4 + moved / (moved < 256 ? 10 : 7);
      if (us < best.us) best = {tile, (int)s, 0, us};
    }
  }
  const int64_t nt = ceil_div(N, 256), tiles = ceil_div(M, 256) * nt, over = tiles % 256;
  if (may_cut && tiles > 256 && over > 0 && over <= 128) {
    const int64_t cut = (tiles - over) / nt * 256;   // whole rows of tiles
    if (cut == 0) return best;
    const double us = tile_rounds_us(f32, 256, cut / 256 * nt, (double)K) + 4 + choose_tile(f32, M - cut, N, K, false).us;
    if (us < best.us) best = {256, 1, cut, us};
  }
  return best;
}

// the product without its first `cut` rows
Product rest_of(int type, Product q, int64_t cut) {
  const int64_t s = (int64_t)dense_type_size(type);
  auto on = [&](const void* p, int64_t ld) { return p ? (const void*)((const char*)p + cut * ld * s) : nullptr; };
  q.A = on(q.A, q.a_across ? 1 : q.lda);
  q.M -= cut;
  q.e.out = (void*)on(q.e.out, q.e.ldo);
  q.e.pre = (void*)on(q.e.pre, q.e.ldp);
  q.e.residual = on(q.e.residual, q.e.ldr);
  return q;
}

// What k_small takes, in us; measured for 1 .. 256 rows and weights of 256^2 .. 4096^2.  Either one workgroup's chain of steps
// along r bounds it (16-bit operands across r come in single values: 43 us at r = 4096, 6 at 1024), or the values that all
// workgroups fetch: 2.2e6 a us in fp32 from L2, 1.5e6 from beyond it (weights of more than 32 MB), 2e6 in 16 bits.
// Where an operand is gated, its gate is computed again in every workgroup that reads it: 0.4 of that rate (4099 rows
// of 515 x 257, fp32 silu: 201 us for both gradients; 62 in tiles).
double small_us(int type, const Product& q, bool gated = false) {
  const int64_t mt = ceil_div(q.M, 16), nt = ceil_div(q.N, 16);
  if (mt * nt > 1 << 20) return 1e30;
  const bool f32 = type == DISN_F32;
  const double K = (double)q.K, values = (double)mt * nt * 32 * K;
  const double chain = f32 ? 0.0027 * K : q.a_across || q.b_across ? 2.5e-6 * K * K : 0.0023 * K;
  const double rate = (f32 ? ((double)q.N * K > 8e6 ? 1.5e6 : 2.2e6) : 2e6) * (gated ? 0.4 : 1.0);
  double us = chain > values / rate ? chain : values / rate;
  const double stores = (double)q.M * q.N / 0.8e6;   // single values
  if (us < stores) us = stores;
  return 2.5 + us;
}
// The same of k_rows_*, up to four rows: W at 6.5 TB/s, and the sum of the parts as a launch more where W lies across r.
// 4096 x 4096 in bf16 / fp32: one row 13.5 / 15.3 us across, 8.8 / 12.6 along r (k_small 43 / 22, 12 / 16; tiles 14 / 32),
// four rows 15.4 / 16.9 and 14.2 / 19.3; eight rows 30 / 21 and 46 / 57, which the other kernels beat.
double rows_us(int type, const Product& q) {
  if (q.a_across || q.M > 4) return 1e30;
  const int64_t size = (int64_t)dense_type_size(type);
  const double read = (double)q.K * q.N * size / 6.5e6;
  if (q.b_across) return 5.5 + read;
  const double chain = 0.6 * q.K / (256 * 16 / size), us = read > chain ? read : chain;
  return q.M > 1 ? 5.5 + 1.4 * us : 3.2 + us;
}

// lanes that share a row of n values, and groups of them along it
int lanes_of(int64_t n, int V) {
  int l = 1;
  while (l < 64 && l * V < n) l *= 2;
  return l;
}
// k_outer writes 4.5 TB/s; the loads of a row's values bound two and three products in 16 bits, and tiles are faster for more
double outer_us(int type, const Product& q) {
  const double results = (double)q.M * q.N;
  if (type == DISN_F32) return q.K <= THIN ? 5 + results / 1.1e6 : 1e30;
  return q.K == 1 ? 5 + results / 2.2e6 : q.K <= 3 ? 5 + results / 1e6 : 1e30;
}
// k_thin and the sum of its parts: the latter's launch, the loads of a row's values of the narrow operand, the wide one
double thin_us(int type, const Product& q) {
  const int64_t S = q.M < q.N ? q.M : q.N, D = q.M < q.N ? q.N : q.M;
  if (type != DISN_F32 || !q.a_across || !q.b_across || S > THIN || D < 4) return 1e30;
  return 13 + 0.8 * S + (double)q.K * (q.M + q.N) / 1.25e6;
}

Plan plan(int type, const Product& q) {
  Plan p{};
  const bool a_across = q.a_across, b_across = q.b_across;
  const int64_t M = q.M, N = q.N, K = q.K;
  if (M == 0 || N == 0 || K == 0) return p;
  const int V = type == DISN_F32 ? 4 : 8, KT = type == DISN_F32 ? KT32 : KT16;
  const bool pack_a = type != DISN_F32 && !tile16_ready(q.A, q.lda), pack_b = type != DISN_F32 && !tile16_ready(q.B, q.ldb);
  const TileChoice c = choose_tile(type == DISN_F32, M, N, K, !pack_a && !pack_b);
  // (a copy of an operand takes 4 us and moves it twice)
  const double tile = c.us + (pack_a ? 4 + 4e-6 * M * K / 4 : 0) + (pack_b ? 4 + 4e-6 * N * K / 4 : 0);
  const double rows = rows_us(type, q), small = small_us(type, q), outer = outer_us(type, q), thin = thin_us(type, q);
  p.us = rows < small ? rows : small;
  if (outer < p.us && outer < tile) {
    p.kind = K_OUTER, p.us = outer;
    return p;
  }
  if (thin < p.us && thin < tile) {
    p.kind = K_THIN, p.us = thin;
    const int64_t D = M < N ? N : M;
    const int lanes = lanes_of(D, V);
    const int64_t groups = ceil_div(D, lanes * V), least = 256 / lanes * 8;   // a step of a workgroup
    p.per = ceil_div(K, ceil_div(512, groups));
    p.per = ceil_div(p.per < least ? least : p.per, least) * least;
    p.splits = (int)ceil_div(K, p.per);
    p.bytes = (size_t)p.splits * M * N * sizeof(float);
    return p;
  }
  if (p.us < tile) {
    p.kind = rows < small ? K_ROWS : K_SMALL;
    if (p.kind == K_SMALL || !b_across) return p;
    const int64_t groups = ceil_div(N, 64 * V);
    int64_t want = ceil_div(1024, groups);
    p.per = ceil_div(ceil_div(K, want), 32) * 32;
    if (p.per > ROWS_MAX_PER) p.per = ROWS_MAX_PER;
    p.splits = (int)ceil_div(K, p.per);
    p.bytes = (size_t)p.splits * M * N * sizeof(float);
    return p;
  }
  p.kind = K_TILE, p.us = tile;
  p.tile = c.tile, p.splits = c.splits, p.cut = c.cut;
  p.per = ceil_div(ceil_div(K, p.splits), KT) * KT;
  p.splits = (int)ceil_div(K, p.per);
  if (p.cut) {   // the two parts run one after the other
    p.bytes = plan(type, rest_of(type, q, p.cut)).bytes;
    return p;
  }
  if (pack_a) p.pack_a = a_across ? pack_bytes(K, M) : pack_bytes(M, K);
  if (pack_b) p.pack_b = b_across ? pack_bytes(K, N) : pack_bytes(N, K);
  p.bytes = p.pack_a + p.pack_b + (p.splits > 1 ? (size_t)p.splits * M * N * sizeof(float) : 0);
  return p;
}

template <typename T>
int launch_finish(DisnCtx* ctx, const float* part, int nparts, int64_t M, int64_t N, const Epilogue& e, hipStream_t stream) {
  if (M == 0 || N == 0) return DISN_OK;
  const int64_t vecs = M * ceil_div(N, Vec<T>::N);
  // with less than 64 / 256 workgroups' worth of results the parts are shared
  if (nparts >= 16 && vecs <= 1 << 14)
    k_finish<T, 16><<<(unsigned)ceil_div(vecs, 16), 256, 0, stream>>>(part, nparts, M, (int)N, e);
  else if (nparts >= 8 && vecs <= 1 << 16)
    k_finish<T, 4><<<(unsigned)ceil_div(vecs, 64), 256, 0, stream>>>(part, nparts, M, (int)N, e);
  else
    k_finish<T, 1><<<(unsigned)(ceil_div(vecs, 256) < 8192 ? ceil_div(vecs, 256) : 8192), 256, 0, stream>>>(part, nparts, M, (int)N, e);
  DISN_HIP(ctx, hipGetLastError());
  return DISN_OK;
}

// LDS of a tile's workgroup
template <typename T, bool A_ACROSS, bool B_ACROSS, int BM, int BN, int THREADS, int RING>
constexpr int tile_lds() {
  if constexpr (sizeof(T) == 4)
    return 2 * (Operand<A_ACROSS, BM, THREADS, 1>::BYTES + Operand<B_ACROSS, BN, THREADS, 1>::BYTES);
  else
    return RING * (BM + BN) * KT16 * 2;
}
// launches a kernel that needs more LDS than a kernel may have unasked; ready: devices that have been asked
int launch_lds(DisnCtx* ctx, std::atomic<uint64_t>& ready, const void* kernel, int64_t blocks, int threads, void** args, int bytes,
               hipStream_t stream) {
  const uint64_t bit = 1ull << (ctx->device & 63);
  if (!(ready.load() & bit)) {
    DISN_HIP(ctx, hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    ready.fetch_or(bit);
  }
  DISN_HIP(ctx, hipLaunchKernel(kernel, dim3((unsigned)blocks), dim3(threads), args, bytes, stream));
  return DISN_OK;
}
int64_t tile_blocks(const TileArgs& a) { return (int64_t)a.mt * a.nt * a.splits; }

template <typename T, bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN, int RING>
int launch_tile(DisnCtx* ctx, TileArgs a, hipStream_t stream) {
  constexpr int THREADS = WM * WN * 64;
  const void* kernel;
  if constexpr (sizeof(T) == 4)   // (a stage of a 128-wide tile is over before the next has come: two under way)
    kernel = (const void*)k_tile32<A_ACROSS, B_ACROSS, BM, BN, WM, WN, BM == 128 ? 2 : 1>;
  else
    kernel = (const void*)k_tile16<T, A_ACROSS, B_ACROSS, BM, BN, WM, WN, RING>;
  static std::atomic<uint64_t> ready{0};
  void* args[] = {&a};
  return launch_lds(ctx, ready, kernel, tile_blocks(a), THREADS, args, tile_lds<T, A_ACROSS, B_ACROSS, BM, BN, THREADS, RING>(), stream);
}
template <typename T, bool W_NK>
int launch_pair(DisnCtx* ctx, TileArgs dx, TileArgs dw, hipStream_t stream) {
  constexpr int x = tile_lds<T, false, W_NK, 128, 128, 256, 4>(), w = tile_lds<T, true, true, 128, 128, 256, 4>();
  static std::atomic<uint64_t> ready{0};
  int split = (int)tile_blocks(dx);
  void* args[] = {&dx, &dw, &split};
  return launch_lds(ctx, ready, (const void*)k_tile_pair<T, W_NK>, split + tile_blocks(dw), 256, args, x > w ? x : w, stream);
}
template <typename T, bool A_ACROSS, bool B_ACROSS>
int launch_tile(DisnCtx* ctx, int tile, const TileArgs& a, hipStream_t stream) {
  if (tile == 256) return launch_tile<T, A_ACROSS, B_ACROSS, 256, 256, 2, 4, 4>(ctx, a, stream);
  if constexpr (sizeof(T) == 2)   // 48 KB of LDS: three a CU
    if (tile_blocks(a) > 512) return launch_tile<T, A_ACROSS, B_ACROSS, 128, 128, 2, 2, 3>(ctx, a, stream);
  return launch_tile<T, A_ACROSS, B_ACROSS, 128, 128, 2, 2, 4>(ctx, a, stream);
}
// a copy of rows x cols values at dst, 16-byte boundaries; *p, *ld become it
template <typename T>
int launch_pack(DisnCtx* ctx, const void** p, int64_t* ld, int64_t rows, int64_t cols, char* dst, hipStream_t stream) {
  const int64_t ldd = ceil_div(cols, 8) * 8, blocks = ceil_div(rows * ldd / 8, 256);
  k_pack<T><<<(unsigned)(blocks < 8192 ? blocks : 8192), 256, 0, stream>>>((const T*)*p, *ld, (T*)dst, ldd, rows, (int)cols);
  DISN_HIP(ctx, hipGetLastError());
  *p = dst, *ld = ldd;
  return DISN_OK;
}

template <typename T, int MR>
void launch_rows(const RowsArgs& a, bool b_across, int splits, hipStream_t stream) {
  if (b_across)
    k_rows_across<T, MR><<<(unsigned)(a.groups * splits), 256, 0, stream>>>(a);
  else
    k_rows_along<T, MR, 4><<<(unsigned)ceil_div(a.N, 4), 256, 0, stream>>>(a);
}

template <typename T>
void launch_outer(const Product& q, hipStream_t stream) {
  OuterArgs a{q.A, q.B, q.a_across ? 1 : q.lda, q.a_across ? q.lda : 1, q.b_across ? 1 : q.ldb, q.b_across ? q.ldb : 1, q.M, 0, (int)q.N, (int)q.K,
              lanes_of(q.N, Vec<T>::N), 0, q.e};
  a.groups = (int)ceil_div(q.N, a.lanes * Vec<T>::N);
  const int64_t step = 256 / a.lanes * 4, most = ceil_div(2048, a.groups);
  a.rows_per = ceil_div(ceil_div(q.M, most), step) * step;
  const unsigned blocks = (unsigned)(ceil_div(q.M, a.rows_per) * a.groups);
  if (q.K == 1) k_outer<T, 1><<<blocks, 256, 0, stream>>>(a);
  else if (q.K <= 4) k_outer<T, 4><<<blocks, 256, 0, stream>>>(a);
  if constexpr (sizeof(T) == 4)
    if (q.K > 4) k_outer<T, THIN><<<blocks, 256, 0, stream>>>(a);
}
void launch_thin(const Product& q, const Plan& p, float* part, hipStream_t stream) {
  const bool a_wide = q.M > q.N;
  ThinArgs a{(const float*)(a_wide ? q.A : q.B), (const float*)(a_wide ? q.B : q.A), a_wide ? q.lda : q.ldb, a_wide ? q.ldb : q.lda, q.K, p.per, (int)(a_wide ? q.M : q.N),
             (int)(a_wide ? q.N : q.M), 0, 0, a_wide ? q.N : 1, a_wide ? 1 : q.N, q.M * q.N, part};
  a.lanes = lanes_of(a.D, 4);
  a.groups = (int)ceil_div(a.D, a.lanes * 4);
  const unsigned blocks = (unsigned)(a.groups * p.splits);
  if (a.S == 1) k_thin<1><<<blocks, 256, 0, stream>>>(a);
  else if (a.S == 2) k_thin<2><<<blocks, 256, 0, stream>>>(a);
  else if (a.S <= 4) k_thin<4><<<blocks, 256, 0, stream>>>(a);
  else k_thin<THIN><<<blocks, 256, 0, stream>>>(a);
}

SmallArgs small_args(const Product& q) {
  SmallArgs s{};
  s.A = {q.A, nullptr, q.lda, 0}, s.B = {q.B, nullptr, q.ldb, 0};
  s.M = (int)q.M, s.N = (int)q.N, s.K = (int)q.K;
  s.mt = (int)ceil_div(q.M, 16), s.nt = (int)ceil_div(q.N, 16);
  s.ks = q.K >= 128 ? SMALL_WAVES : 1;
  s.e = q.e;
  return s;
}
int64_t small_blocks(const SmallArgs& s) { return (int64_t)s.mt * ceil_div(s.nt, SMALL_WAVES / s.ks); }

// a product in tiles: copies what has to be copied and fills in the kernel's arguments
template <typename T>
int prepare_tile(DisnCtx* ctx, Product q, const Plan& p, char* ws, TileArgs* t, hipStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.pack_a) DISN_TRY(launch_pack<T>(ctx, &q.A, &q.lda, q.a_across ? q.K : q.M, q.a_across ? q.M : q.K, ws, stream));
    if (p.pack_b) DISN_TRY(launch_pack<T>(ctx, &q.B, &q.ldb, q.b_across ? q.K : q.N, q.b_across ? q.N : q.K, ws + p.pack_a, stream));
  }
  *t = {q.A, q.B, q.lda, q.ldb, (int)q.M, (int)q.N, q.K, p.per, (int)ceil_div(q.M, p.tile), (int)ceil_div(q.N, p.tile), p.splits,
        (float*)(ws + p.pack_a + p.pack_b), q.e};
  return DISN_OK;
}

// one product by its plan; ws: plan.bytes of workspace
template <typename T>
int run_product(DisnCtx* ctx, Product q, Plan p, char* ws, hipStream_t stream) {
  if (p.cut) {
    const Product rest = rest_of(sizeof(T) == 4 ? DISN_F32 : DISN_BF16, q, p.cut);
    DISN_TRY(run_product<T>(ctx, rest, plan(sizeof(T) == 4 ? DISN_F32 : DISN_BF16, rest), ws, stream));
    q.M = p.cut;
    p.cut = 0;
  }
  float* part = (float*)ws;
  if (q.M == 0 || q.N == 0) return DISN_OK;
  if (p.kind == K_EMPTY) return launch_finish<T>(ctx, nullptr, 0, q.M, q.N, q.e, stream);
  if (p.kind == K_SMALL) {
    const SmallArgs s = small_args(q);
    const unsigned blocks = (unsigned)small_blocks(s);
    if (q.a_across) {
      // dW beside a large dx: the paired kernel without a dx
      k_small_backward<T, false><<<blocks, SMALL_WAVES * 64, 0, stream>>>(s, s, 0);
    } else if (q.b_across) {
      k_small<T, true><<<blocks, SMALL_WAVES * 64, 0, stream>>>(s);
    } else {
      k_small<T, false><<<blocks, SMALL_WAVES * 64, 0, stream>>>(s);
    }
    DISN_HIP(ctx, hipGetLastError());
    return DISN_OK;
  }
  if (p.kind == K_OUTER) {
    launch_outer<T>(q, stream);
    DISN_HIP(ctx, hipGetLastError());
    return DISN_OK;
  }
  if (p.kind == K_THIN) {
    launch_thin(q, p, part, stream);
    DISN_HIP(ctx, hipGetLastError());
    return launch_finish<T>(ctx, part, p.splits, q.M, q.N, q.e, stream);
  }
  if (p.kind == K_ROWS) {
    RowsArgs r{q.A, q.B, q.lda, q.ldb, (int)q.M, (int)q.N, (int)q.K, (int)p.per, (int)ceil_div(q.N, 64 * Vec<T>::N), part, q.e};
    if (q.M == 1) launch_rows<T, 1>(r, q.b_across, p.splits, stream);
    else launch_rows<T, 4>(r, q.b_across, p.splits, stream);
    DISN_HIP(ctx, hipGetLastError());
    return q.b_across ? launch_finish<T>(ctx, part, p.splits, q.M, q.N, q.e, stream) : DISN_OK;
  }
  TileArgs t;
  DISN_TRY(prepare_tile<T>(ctx, q, p, ws, &t, stream));
  if (q.a_across) DISN_TRY((launch_tile<T, true, true>(ctx, p.tile, t, stream)));
  else if (q.b_across) DISN_TRY((launch_tile<T, false, true>(ctx, p.tile, t, stream)));
  else DISN_TRY((launch_tile<T, false, false>(ctx, p.tile, t, stream)));
  return p.splits > 1 ? launch_finish<T>(ctx, t.part, p.splits, q.M, q.N, q.e, stream) : DISN_OK;
}

// ---- host: arguments -----------------------------------------------------------------------------------------------------
// n and k are bounded by the 32-bit offsets of a tile's operands (tile16_ready; a copy's rows are as long as n or k) and by
// the grids of k_rows_along and k_sum_partials
bool linear_size_ok(int64_t v) { return v >= 0 && v <= DISN_LINEAR_MAX; }
int check_linear(DisnCtx* ctx, const DisnLinear* a) {
  const char* f = "disn_linear";
  if (!a) return disn_fail(ctx, DISN_E_ARG, "%s: null arguments", f);
  if (!dense_type_ok(a->type) || a->act < DISN_ACT_NONE || a->act > DISN_ACT_SILU || a->w_nk < 0 || a->w_nk > 1 || a->reserved)
    return disn_fail(ctx, DISN_E_ARG, "%s: bad type %d, act %d, w_nk %d or reserved field", f, a->type, a->act, a->w_nk);
  if (!dense_size_ok(a->m) || !linear_size_ok(a->n) || !linear_size_ok(a->k))
    return disn_fail(ctx, DISN_E_ARG, "%s: sizes m %lld, n %lld, k %lld (n and k up to %d)", f, (long long)a->m, (long long)a->n,
                     (long long)a->k, DISN_LINEAR_MAX);
  const size_t s = dense_type_size(a->type);
  if (a->m == 0 || a->n == 0) return DISN_OK;
  if (!dense_matrix_ok(a->x, a->m, a->k, a->ldx, s, true) ||
      !dense_matrix_ok(a->w, a->w_nk ? a->n : a->k, a->w_nk ? a->k : a->n, a->ldw, s, true) ||
      !dense_matrix_ok(a->y, a->m, a->n, a->ldy, s, false) || (a->residual && !dense_matrix_ok(a->residual, a->m, a->n, a->ldr, s, true)) ||
      (a->pre && !dense_matrix_ok(a->pre, a->m, a->n, a->ldp, s, false)))
    return disn_fail(ctx, DISN_E_ARG, "%s: a matrix is null, misaligned or has a bad row distance", f);
  if (!dense_aligned(a->bias, s)) return disn_fail(ctx, DISN_E_ARG, "%s: bias is misaligned", f);
  return DISN_OK;
}

int check_linear_grad(DisnCtx* ctx, const DisnLinearGrad* a) {
  const char* f = "disn_linear_backward";
  if (!a) return disn_fail(ctx, DISN_E_ARG, "%s: null arguments", f);
  if (!dense_type_ok(a->type) || a->act < DISN_ACT_NONE || a->act > DISN_ACT_SILU || a->w_nk < 0 || a->w_nk > 1 || a->reserved)
    return disn_fail(ctx, DISN_E_ARG, "%s: bad type %d, act %d, w_nk %d or reserved field", f, a->type, a->act, a->w_nk);
  if (!dense_size_ok(a->m) || !linear_size_ok(a->n) || !linear_size_ok(a->k))
    return disn_fail(ctx, DISN_E_ARG, "%s: sizes m %lld, n %lld, k %lld (n and k up to %d)", f, (long long)a->m, (long long)a->n,
                     (long long)a->k, DISN_LINEAR_MAX);
  const size_t s = dense_type_size(a->type);
  const int64_t wr = a->w_nk ? a->n : a->k, wc = a->w_nk ? a->k : a->n;
  if ((a->act == DISN_ACT_NONE) != !a->pre && a->m && a->n)
    return disn_fail(ctx, DISN_E_ARG, "%s: pre belongs to an activation (act %d)", f, a->act);
  if (!dense_matrix_ok(a->dy, a->m, a->n, a->lddy, s, true) || (a->pre && !dense_matrix_ok(a->pre, a->m, a->n, a->ldp, s, true)) ||
      (a->dx && !dense_matrix_ok(a->dx, a->m, a->k, a->lddx, s, false)) || (a->dw && !dense_matrix_ok(a->dw, wr, wc, a->lddw, s, false)) ||
      (a->dx && !dense_matrix_ok(a->w, wr, wc, a->ldw, s, true)) || (a->dw && !dense_matrix_ok(a->x, a->m, a->k, a->ldx, s, true)))
    return disn_fail(ctx, DISN_E_ARG, "%s: a matrix is null, misaligned or has a bad row distance", f);
  if (!dense_aligned(a->db, s)) return disn_fail(ctx, DISN_E_ARG, "%s: db is misaligned", f);
  return DISN_OK;
}

// Whether results are stored past the caches.  A line that stores of two waves fill goes out in parts then: rows of whole lines
// (30000 x 304, relu, fp16: 1056 results a row 43.4 -> 42.1 us, but 1000 of them 42 -> 49), or more bytes than the last cache holds
// anyway (fp32, 1000 results a row with a residual, 240 MB: 163 -> 136 us; without, 120 MB: 116 -> 121; fp16 with a residual
// and z, 180 MB: 64 -> 73).
int streams(int type, const Product& q) {
  const Epilogue& e = q.e;
  const int64_t size = (int64_t)dense_type_size(type), matrices = 1 + (e.pre != nullptr) + (e.residual != nullptr);
  auto whole = [&](const void* p, int64_t ld) { return !p || (dense_aligned(p, 64) && ld * size % 64 == 0); };
  return (whole(e.out, e.ldo) && whole(e.pre, e.ldp)) || q.M * q.N * size * matrices > 200000000;
}
Product forward_product(const DisnLinear* a) {
  Product q{a->x, a->w, a->ldx, a->ldw, false, a->w_nk == 0, a->m, a->n, a->k,
            {a->bias, a->residual, a->pre, a->y, a->ldr, a->ldp, a->ldy, a->act, 0}};
  q.e.stream = streams(a->type, q);
  return q;
}

// The backward pass of one call: small ones are one launch; others write dz once (act != none), then two products, at once
// where they fit the chip together.
struct GradPlan {
  bool small, pair;
  Plan dx, dw;
  int64_t ldz, gate_blocks, gate_rows;
  int gate_lanes, gate_groups;
  size_t off_sums, off_part, bytes;   // workspace: dz, partial column sums, partial products
};
// the two products on dz as it lies at (dz, ldz)
void grad_products(const DisnLinearGrad* a, const void* dz, int64_t ldz, Product* dx, Product* dw) {
  *dx = {dz, a->w, ldz, a->ldw, false, a->w_nk != 0, a->m, a->k, a->n, {nullptr, nullptr, nullptr, a->dx, 0, 0, a->lddx, DISN_ACT_NONE, 0}};
  *dw = {a->x, dz, a->ldx, ldz, true, true, a->k, a->n, a->m, {nullptr, nullptr, nullptr, a->dw, 0, 0, a->lddw, DISN_ACT_NONE, 0}};
  dx->e.stream = streams(a->type, *dx), dw->e.stream = streams(a->type, *dw);
  if (a->w_nk) *dw = {dz, a->x, ldz, a->ldx, true, true, a->n, a->k, a->m, dw->e};
}
GradPlan plan_backward(const DisnLinearGrad* a) {
  GradPlan g{};
  const size_t s = dense_type_size(a->type);
  Product dx, dw;
  g.ldz = ceil_div(a->n, 8) * 8;
  // dz of an activation will lie in the workspace, at an address like 256
  if (a->act != DISN_ACT_NONE) grad_products(a, (const void*)256, g.ldz, &dx, &dw);
  else grad_products(a, a->dy, a->lddy, &dx, &dw);
  if (a->dx) g.dx = plan(a->type, dx);
  if (a->dw) g.dw = plan(a->type, dw);
  // both products at once where they are 128-wide tiles that fit the chip together, two a CU
  auto blocks128 = [](const Plan& p, const Product& q) {
    return p.kind == K_TILE && p.tile == 128 && !p.cut ? ceil_div(q.M, 128) * ceil_div(q.N, 128) * p.splits : 1 << 30;
  };
  g.pair = a->dx && a->dw && blocks128(g.dx, dx) + blocks128(g.dw, dw) <= 512;
  // one launch of k_small_backward, or dz and the bias's gradient first (two launches, 8 us and dz written and read)
  const bool gated = a->act != DISN_ACT_NONE;
  const double products = !g.pair ? g.dx.us + g.dw.us : g.dx.us > g.dw.us ? g.dx.us + 3 : g.dw.us + 3;
  const double apart = products + 8 + 3e-6 * a->m * a->n * s / 5;
  g.small = a->m && a->n && a->k && a->dw && (a->dx ? small_us(a->type, dx, gated) : 0) + small_us(a->type, dw, gated) <= apart;
  if (g.small) return g;
  const int V = a->n < (int64_t)(16 / s) ? 1 : (int)(16 / s);
  g.gate_lanes = lanes_of(a->n, V);
  g.gate_groups = (int)ceil_div(a->n, g.gate_lanes * V);
  if (g.gate_groups < 1) g.gate_groups = 1;
  // row blocks: about 1024 workgroups, at least 4 rows a thread
  const int64_t lines = 256 / g.gate_lanes;
  int64_t blocks = ceil_div(1024, g.gate_groups);
  if (blocks > ceil_div(a->m, lines * 4)) blocks = ceil_div(a->m, lines * 4);
  if (blocks < 1) blocks = 1;
  g.gate_rows = ceil_div(a->m, blocks);
  g.gate_blocks = a->m ? ceil_div(a->m, g.gate_rows) : 0;
  size_t at = 0;
  if (a->act != DISN_ACT_NONE && (a->dx || a->dw)) at += align256((size_t)a->m * g.ldz * s);
  g.off_sums = at;
  if (a->db) at += align256((size_t)g.gate_blocks * a->n * sizeof(float));
  g.off_part = at;
  at += g.pair ? align256(g.dx.bytes) + g.dw.bytes : g.dx.bytes > g.dw.bytes ? g.dx.bytes : g.dw.bytes;
  g.bytes = at;
  return g;
}

template <typename T>
int run_backward(DisnCtx* ctx, const DisnLinearGrad* a, const GradPlan& g, char* ws, hipStream_t stream) {
  const bool gated = a->act != DISN_ACT_NONE;
  const void* dz = a->dy;
  int64_t ldz = a->lddy;
  if (!g.small) {
    const bool write = gated && (a->dx || a->dw);
    if (a->n && a->m && (write || a->db)) {
      GateArgs k{a->dy, a->pre, write ? ws : nullptr, a->db ? (float*)(ws + g.off_sums) : nullptr, a->lddy, a->ldp, g.ldz, a->m,
                 g.gate_rows, (int)a->n, g.gate_lanes, g.gate_groups, a->act};
      const unsigned blocks = (unsigned)(g.gate_groups * g.gate_blocks);
      if (a->n < Vec<T>::N) k_gate<T, true><<<blocks, 256, 0, stream>>>(k);
      else k_gate<T, false><<<blocks, 256, 0, stream>>>(k);
      DISN_HIP(ctx, hipGetLastError());
    }
    if (a->db && a->n) {
      k_sum_partials<T><<<(unsigned)ceil_div(a->n, 16), 256, 0, stream>>>((const float*)(ws + g.off_sums), (int)g.gate_blocks, a->n, a->n,
                                                                          (T*)a->db, (T*)nullptr);
      DISN_HIP(ctx, hipGetLastError());
    }
    if (write) dz = ws, ldz = g.ldz;
  }
  Product dx, dw;
  grad_products(a, dz, ldz, &dx, &dw);
  if (g.pair) {
    TileArgs tx, tw;
    DISN_TRY(prepare_tile<T>(ctx, dx, g.dx, ws + g.off_part, &tx, stream));
    DISN_TRY(prepare_tile<T>(ctx, dw, g.dw, ws + g.off_part + align256(g.dx.bytes), &tw, stream));
    if (a->w_nk) DISN_TRY((launch_pair<T, true>(ctx, tx, tw, stream)));
    else DISN_TRY((launch_pair<T, false>(ctx, tx, tw, stream)));
    if (g.dx.splits > 1) DISN_TRY(launch_finish<T>(ctx, tx.part, g.dx.splits, dx.M, dx.N, dx.e, stream));
    if (g.dw.splits > 1) DISN_TRY(launch_finish<T>(ctx, tw.part, g.dw.splits, dw.M, dw.N, dw.e, stream));
    return DISN_OK;
  }
  if (!g.small) {
    if (a->dx) DISN_TRY(run_product<T>(ctx, dx, g.dx, ws + g.off_part, stream));
    if (a->dw) DISN_TRY(run_product<T>(ctx, dw, g.dw, ws + g.off_part, stream));
    return DISN_OK;
  }
  SmallArgs sx = small_args(dx), sw = small_args(dw);
  sx.act = sw.act = a->act;
  sx.A.gate = a->pre, sx.A.ldg = a->ldp;
  SmallOperand& of = a->w_nk ? sw.A : sw.B;
  of.gate = a->pre, of.ldg = a->ldp;
  sw.rsum = a->db, sw.rsum_of_a = a->w_nk;
  const int64_t first = a->dx ? small_blocks(sx) : 0, blocks = first + small_blocks(sw);
  if (a->w_nk)
    k_small_backward<T, true><<<(unsigned)blocks, SMALL_WAVES * 64, 0, stream>>>(sx, sw, (int)first);
  else
    k_small_backward<T, false><<<(unsigned)blocks, SMALL_WAVES * 64, 0, stream>>>(sx, sw, (int)first);
  DISN_HIP(ctx, hipGetLastError());
  return DISN_OK;
}

}  // namespace

extern "C" int disn_linear_workspace(DisnCtx* ctx, const DisnLinear* a, size_t* bytes) {
  if (!ctx) return DISN_E_ARG;
  if (!bytes) return disn_fail(ctx, DISN_E_ARG, "disn_linear_workspace: null result");
  DISN_TRY(check_linear(ctx, a));
  *bytes = plan(a->type, forward_product(a)).bytes;
  return DISN_OK;
}

extern "C" int disn_linear(DisnCtx* ctx, const DisnLinear* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!ctx) return DISN_E_ARG;
  DISN_TRY(check_linear(ctx, a));
  const Plan p = plan(a->type, forward_product(a));
  if (p.bytes && (!workspace || !dense_aligned(workspace, 16) || workspace_bytes < p.bytes))
    return disn_fail(ctx, DISN_E_ARG, "disn_linear: needs %zu bytes of 16-byte aligned workspace", p.bytes);
  DISN_HIP(ctx, hipSetDevice(ctx->device));
  return dense_dispatch(a->type, [&](auto t) {
    return run_product<decltype(t)>(ctx, forward_product(a), p, (char*)workspace, (hipStream_t)stream);
  });
}

extern "C" int disn_linear_backward_workspace(DisnCtx* ctx, const DisnLinearGrad* a, size_t* bytes) {
  if (!ctx) return DISN_E_ARG;
  if (!bytes) return disn_fail(ctx, DISN_E_ARG, "disn_linear_backward_workspace: null result");
  DISN_TRY(check_linear_grad(ctx, a));
  *bytes = plan_backward(a).bytes;
  return DISN_OK;
}

extern "C" int disn_linear_backward(DisnCtx* ctx, const DisnLinearGrad* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!ctx) return DISN_E_ARG;
  DISN_TRY(check_linear_grad(ctx, a));
  const GradPlan g = plan_backward(a);
  if (g.bytes && (!workspace || !dense_aligned(workspace, 16) || workspace_bytes < g.bytes))
    return disn_fail(ctx, DISN_E_ARG, "disn_linear_backward: needs %zu bytes of 16-byte aligned workspace", g.bytes);
  DISN_HIP(ctx, hipSetDevice(ctx->device));
  return dense_dispatch(a->type, [&](auto t) {
    return run_backward<decltype(t)>(ctx, a, g, (char*)workspace, (hipStream_t)stream);
  });
}
