// norm.hip -- layer norm over the rows of a matrix, forward and backward (include/disn.h).
//
// Forward, per row:   mean = sum x / d;  var = sum (x - mean)^2 / d;  rstd = 1 / sqrt(var + eps);
//                     y = (x - mean) rstd g + b
// Backward, per row:  h = (x - mean) rstd;  t = dy g;  dx = rstd (t - avg(t) - h avg(t h)) + residual
//            columns: dg = sum over rows of dy h;  db = sum over rows of dy
//
// Both are bound by memory: every value is read once and written once.  A group of G threads holds a whole row in
// registers, E values a thread in 16-byte pieces, so the variance is the sum of squared distances from the mean that
// is already known (not a difference of two large sums) and costs no second read.  G up to 64: rows inside a wave
// (no barrier, sums by lane exchange), 256 / 512: a row per workgroup.  The backward pass walks over rows with a
// fixed set of workgroups; a thread meets the same columns in every row and sums their dg, db in registers; the
// workgroups' sums are added in order by a second kernel.  Few waves fit beside these registers, so each reads its next
// row while it works on the present one (us without / with, 300 MB of bf16 rows: d = 768 343 / 167, 1024 276 / 168,
// 4096 300 / 189); so does the forward pass of the longest rows (d = 5000 168 / 127).
// Measured: 262144 x 512 bf16 forward 106 us (5.1 TB/s of what is read and written), backward with a residual 194 us (5.5), 5003 x 1537
// fp32 backward 25 us (3.7).  Rows of 16-bit values that start at odd places are slower:
// 300 MB in rows of 1031 forward 198 us, backward 325; of 1024 114 and 176 (read as aligned dwords and shifted 182 and 357,
// stored in three aligned pieces 213 and 336).
#include "dense.h"

namespace {

struct NormArgs {
  const void *x, *weight, *bias, *dy, *residual;
  const float *mean_in, *rstd_in;
  void *y, *dweight, *dbias;
  float *mean, *rstd, *part;
  int64_t ldx, ldy, lddy, ldr;
  int64_t rows;
  int d;
  float eps;
};

// sum over the G threads of a row's group; lds: two slots of 16 floats, used in turn (a slot is rewritten two sums
// later, behind the other sum's barrier)
template <int G>
__device__ __forceinline__ float group_sum(float v, float (*lds)[16], int slot) {
#pragma unroll
  for (int m = (G < 64 ? G : 64) / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  if constexpr (G > 64) {
    if ((threadIdx.x & 63) == 0) lds[slot][threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[slot][0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) v += lds[slot][i];
  }
  return v;
}

// column of the piece p that a thread of a group holds, and how many of its values lie inside the row
template <typename T, int G>
__device__ __forceinline__ int piece_col(int t, int p) { return (p * G + t) * Vec<T>::N; }

template <typename T, int E>
__device__ __forceinline__ void widen(const Vec<T> (&in)[E / Vec<T>::N], float (&out)[E]) {
#pragma unroll
  for (int i = 0; i < E; ++i) out[i] = (float)in[i / Vec<T>::N].v[i % Vec<T>::N];
}

// How the end of a row is met.  WHOLE: rows of whole pieces.  SHIFT: the piece that holds a row's end is read from further in
// front (its other values lie in the same row) and shifted once it is there, so that no load waits in a branch.  SHORT: rows
// of less than one piece.
enum Ends { WHOLE, SHIFT, SHORT };

template <typename T, int G, int E, Ends ENDS>
struct Row {
  static constexpr int N = Vec<T>::N, P = E / N;
  int at[P], back[P];   // column each piece is read from; by how many values it is shifted then (N: all of it)
  bool any;             // whether this wave shifts
  __device__ __forceinline__ Row(int t, int d) {
    any = false;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = piece_col<T, G>(t, p);
      back[p] = c >= d ? N : c + N > d ? c + N - d : 0;
      at[p] = ENDS == SHIFT && c < d ? c - back[p] : c < d ? c : 0;
      any |= back[p] != 0;
    }
    if (ENDS == SHIFT) any = __any(any);
  }
  __device__ __forceinline__ void load(const T* row, Vec<T> (&out)[P]) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (ENDS == SHIFT) out[p] = load_vec(row + at[p]);
      else if (ENDS == WHOLE) out[p] = back[p] ? Vec<T>{} : load_vec(row + at[p]);
      else out[p] = load_vec(row + at[p], N - back[p], 0);
    }
  }
  // zeros behind the row's end
  __device__ __forceinline__ void settle(Vec<T> (&out)[P]) const {
    if (ENDS != SHIFT || !any) return;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      uint32_t w[4];
      __builtin_memcpy(w, &out[p], 16);
      const int bits = back[p] * 8 * (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bits & 64 ? (i < 2 ? w[i + 2] : 0) : w[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bits & 32 ? (i < 3 ? w[i + 1] : 0) : w[i];
      if (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bits & 16 ? (w[i] >> 16) | (i < 3 ? w[i + 1] << 16 : 0) : w[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = bits & 128 ? 0 : w[i];
      __builtin_memcpy(&out[p], w, 16);
    }
  }
};

// Whether all values of a row are equal: their mean is that value then, so that the row gives the bias (and 0 / 0 without an
// eps).  A sum of equal fp32 values is rounded, and its mean may be some steps off; one of up to 8192 16-bit values is exact, so
// there is nothing to do for those.  Waves that share a row leave their verdict in the upper half of the sum's slot.
template <typename T, int G, int E>
struct Equal {
  float first;   // a value of the row
  bool other;    // whether this group of lanes has met another
  __device__ __forceinline__ Equal(const float (&x)[E], int t, int d, float* slot) {
    if constexpr (sizeof(T) == 4) {
      const int lane = threadIdx.x & 63, base = G < 64 ? lane & ~(G - 1) : 0;   // (every wave's first lane holds values of the row)
      first = __shfl(x[0], base, 64);
      bool o = false;
#pragma unroll
      for (int i = 0; i < E; ++i) o |= piece_col<T, G>(t, i / Vec<T>::N) + i % Vec<T>::N < d && x[i] != first;
      const uint64_t met = __ballot(o) >> base;
      other = (G < 64 ? met & ((1ull << (G & 63)) - 1) : met) != 0;
      if (G > 64 && lane == 0) slot[8 + (threadIdx.x >> 6)] = other ? __builtin_nanf("") : first;
    }
  }
  // behind the sum's barrier
  __device__ __forceinline__ float mean_or(float mean, const float* slot) const {
    if constexpr (sizeof(T) == 4) {
      bool all = !other;
      if constexpr (G > 64) {
        all = true;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) all &= slot[8 + i] == slot[8];   // (a NaN is not equal to itself)
        return all ? slot[8] : mean;
      }
      return all ? first : mean;
    }
    return mean;
  }
};

template <typename T, int G, int E, Ends ENDS>
__global__ __launch_bounds__(G <= 64 ? 256 : G) void k_layer_norm(NormArgs a) {
  constexpr int N = Vec<T>::N, P = E / N, B = G <= 64 ? 256 : G;
  __shared__ float lds[2][16];
  const int t = threadIdx.x % G, d = a.d;
  const Row<T, G, E, ENDS> ends(t, d);
  float w[E], b[E];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = piece_col<T, G>(t, p), n = c < d ? d - c : 0;
    const Vec<T> wv = a.weight ? load_vec((const T*)a.weight + (n ? c : 0), n, c) : Vec<T>{};
    const Vec<T> bv = a.bias ? load_vec((const T*)a.bias + (n ? c : 0), n, c) : Vec<T>{};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[p * N + i] = a.weight ? (float)wv.v[i] : 1.0f;
      b[p * N + i] = a.bias ? (float)bv.v[i] : 0.0f;
    }
  }
  const float inv = 1.0f / (float)d;
  constexpr bool AHEAD = G == 512;   // the next row is read early
  const int64_t step = (int64_t)gridDim.x * (B / G);
  int64_t row = (int64_t)blockIdx.x * (B / G) + threadIdx.x / G;
  Vec<T> next[P];
  if (AHEAD) ends.load((const T*)a.x + row * a.ldx, next);   // (no more workgroups than rows)
  for (; row < a.rows; row += step) {
    Vec<T> xv[P];
    if (AHEAD) {
#pragma unroll
      for (int p = 0; p < P; ++p) xv[p] = next[p];
      ends.load((const T*)a.x + min(row + step, a.rows - 1) * a.ldx, next);
    } else {
      ends.load((const T*)a.x + row * a.ldx, xv);
    }
    ends.settle(xv);
    float x[E];
    widen<T, E>(xv, x);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) s += x[i];   // places behind the row hold 0
    const Equal<T, G, E> equal(x, t, d, lds[0]);
    const float mean = equal.mean_or(group_sum<G>(s, lds, 0) / (float)d, lds[0]);
    s = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float c = piece_col<T, G>(t, p) + i < d ? x[p * N + i] - mean : 0.0f;
        x[p * N + i] = c;
        s = fmaf(c, c, s);
      }
    const float rstd = 1.0f / sqrtf(group_sum<G>(s, lds, 1) * inv + a.eps);
    if (t == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = (T*)a.y + row * a.ldy;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = piece_col<T, G>(t, p);
      if (c >= d) break;
      Vec<T> o;
#pragma unroll
      for (int i = 0; i < N; ++i) x[p * N + i] = fmaf(x[p * N + i] * rstd, w[p * N + i], b[p * N + i]);
      narrow<T, N>(x + p * N, o.v);
      store_vec<T, true>(y + c, o, ENDS == WHOLE ? N : d - c);
    }
  }
}

template <typename T, int G, int E, Ends ENDS>
__global__ __launch_bounds__(G <= 64 ? 256 : G) void k_layer_norm_backward(NormArgs a) {
  constexpr int N = Vec<T>::N, P = E / N, B = G <= 64 ? 256 : G;
  __shared__ float lds[2][16];
  const int t = threadIdx.x % G, d = a.d;
  const Row<T, G, E, ENDS> ends(t, d);
  float w[E], dg[E], db[E];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = piece_col<T, G>(t, p), n = c < d ? d - c : 0;
    const Vec<T> wv = a.weight ? load_vec((const T*)a.weight + (n ? c : 0), n, c) : Vec<T>{};
#pragma unroll
    for (int i = 0; i < N; ++i) w[p * N + i] = a.weight ? (float)wv.v[i] : 1.0f;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) dg[i] = db[i] = 0.0f;
  const float inv = 1.0f / (float)d;
  Vec<T> next_x[P], next_g[P], next_r[P];
  float next_mean, next_rstd;
  auto fetch = [&](int64_t row) {
    row = min(row, a.rows - 1);
    ends.load((const T*)a.x + row * a.ldx, next_x);
    ends.load((const T*)a.dy + row * a.lddy, next_g);
    if (a.y && a.residual) ends.load((const T*)a.residual + row * a.ldr, next_r);
    next_mean = a.mean_in[row], next_rstd = a.rstd_in[row];
  };
  const int64_t step = (int64_t)gridDim.x * (B / G);
  int64_t row = (int64_t)blockIdx.x * (B / G) + threadIdx.x / G;
  if (a.rows > 0) fetch(row);
  for (; row < a.rows; row += step) {
    Vec<T> xv[P], gv[P], rv[P];
#pragma unroll
    for (int p = 0; p < P; ++p) xv[p] = next_x[p], gv[p] = next_g[p], rv[p] = next_r[p];
    const float mean = next_mean, rstd = next_rstd;
    fetch(row + step);
    ends.settle(xv);
    ends.settle(gv);
    if (a.y && a.residual) ends.settle(rv);
    float h[E], g[E], s1 = 0.0f, s2 = 0.0f;
    widen<T, E>(xv, h);
    widen<T, E>(gv, g);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      h[i] = (h[i] - mean) * rstd;   // places behind the row: finite or not, their g is 0 ...
      const bool in = piece_col<T, G>(t, i / N) + i % N < d;
      if (!in) h[i] = 0.0f;          // ... and a NaN of the row's statistics must not meet it
      dg[i] = fmaf(g[i], h[i], dg[i]);
      db[i] += g[i];
      g[i] *= w[i];
      s1 += g[i];
      s2 = fmaf(g[i], h[i], s2);
    }
    if (!a.y) continue;
    s1 = group_sum<G>(s1, lds, 0) * inv;
    s2 = group_sum<G>(s2, lds, 1) * inv;
    T* dx = (T*)a.y + row * a.ldy;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = piece_col<T, G>(t, p);
      if (c >= d) break;
      Vec<T> o;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int e = p * N + i;
        float v = rstd * (g[e] - s1 - h[e] * s2);
        if (a.residual) v += (float)rv[p].v[i];
        g[e] = v;
      }
      narrow<T, N>(g + p * N, o.v);
      store_vec<T, true>(dx + c, o, ENDS == WHOLE ? N : d - c);
    }
  }
  if (!a.dweight && !a.dbias) return;
  // the workgroup's sums: the groups of a wave by lane exchange, four waves through LDS, then out (one workgroup) or partial sums
  constexpr int WAVES = G <= 64 ? 4 : 1;
  __shared__ float red[WAVES > 1 ? WAVES * G * E : 1];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&v)[E] = which ? db : dg;
    if constexpr (WAVES > 1) {
      if (which) __syncthreads();
#pragma unroll
      for (int i = 0; i < E; ++i) {
#pragma unroll
        for (int m = G; m < 64; m <<= 1) v[i] += __shfl_xor(v[i], m, 64);
        if ((threadIdx.x & 63) < G) red[((threadIdx.x >> 6) * G + t) * E + i] = v[i];
      }
      __syncthreads();
      if (threadIdx.x < G) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (red[t * E + i] + red[(G + t) * E + i]) + (red[(2 * G + t) * E + i] + red[(3 * G + t) * E + i]);
      }
    }
    if (threadIdx.x < G) {
      T* out = (T*)(which ? a.dbias : a.dweight);
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = piece_col<T, G>(t, p) + i;
          if (c >= d) continue;
          if (gridDim.x == 1) {
            if (out) out[c] = (T)v[p * N + i];
          } else {
            a.part[(size_t)blockIdx.x * 2 * d + (size_t)which * d + c] = v[p * N + i];
          }
        }
    }
  }
}

// Group size and values per thread for a row of d values: the smallest group that holds it, 8 values a thread, up to a
// wave (lanes without values cost time: 16-bit rows of 40 in groups of 8 / 16 136 / 212 us, rows of 200 in groups of 32 / 64
// 130 / 183); 16 a thread before a row is spread over more waves.
struct NormShape {
  int group, per_thread;
};
NormShape norm_shape(int64_t d) {
  if (d <= 512) return {d <= 64 ? 8 : d <= 128 ? 16 : d <= 256 ? 32 : 64, 8};
  if (d <= 1024) return {64, 16};
  if (d <= 2048) return {256, 8};
  if (d <= 4096) return {256, 16};
  return {512, 16};
}
int64_t norm_rows_at_once(const NormShape& s) { return s.group <= 64 ? 256 / s.group : 1; }
// Workgroups of the backward pass: what the chip holds of them at once, each at least two rows a group, so that the partial
// sums (2 d floats a workgroup) stay small beside the rows it reads.
// Measured in us at 256 / 512 / 768 / 1024 workgroups, 300 MB of rows: 512 bf16 253 / 170 / 161 / 171 and fp32
// 244 / 167 / 175 / 176, 1024 bf16 172 / 168 / 181 / 202, 2000 bf16 496 / 270 / 216 / 195 and fp32 270 / 170 / 173 / 183, 1100
// fp32 432 / 240 / 190 / 174, 3001 bf16 393 / 282 / 323 / 295, 5000 bf16 265 / 274 / 284 / 292.
int64_t norm_backward_grid(const NormShape& s, int type, int64_t rows) {
  const int64_t per = norm_rows_at_once(s), want = (rows + per * 2 - 1) / (per * 2);
  const int64_t most = s.group == 512 ? 256 : s.per_thread > 8 ? 512 : s.group == 256 && type != DISN_F32 ? 1024 : 768;
  return want < 1 ? 1 : want < most ? want : most;
}

template <typename T, int G, int E>
void launch_norm(bool backward, const NormArgs& a, int64_t grid, hipStream_t stream) {
  constexpr int B = G <= 64 ? 256 : G;
  const int N = Vec<T>::N;
  const Ends ends = a.d % N == 0 ? WHOLE : a.d > N ? SHIFT : SHORT;
  if constexpr (G == 8)
    if (ends == SHORT) {
      if (backward) k_layer_norm_backward<T, G, E, SHORT><<<(unsigned)grid, B, 0, stream>>>(a);
      else k_layer_norm<T, G, E, SHORT><<<(unsigned)grid, B, 0, stream>>>(a);
      return;
    }
  if (backward && ends == WHOLE) k_layer_norm_backward<T, G, E, WHOLE><<<(unsigned)grid, B, 0, stream>>>(a);
  else if (backward) k_layer_norm_backward<T, G, E, SHIFT><<<(unsigned)grid, B, 0, stream>>>(a);
  else if (ends == WHOLE) k_layer_norm<T, G, E, WHOLE><<<(unsigned)grid, B, 0, stream>>>(a);
  else k_layer_norm<T, G, E, SHIFT><<<(unsigned)grid, B, 0, stream>>>(a);
}
template <typename T>
void launch_norm(const NormShape& s, bool backward, const NormArgs& a, int64_t grid, hipStream_t stream) {
  if (s.group == 8) launch_norm<T, 8, 8>(backward, a, grid, stream);
  else if (s.group == 16) launch_norm<T, 16, 8>(backward, a, grid, stream);
  else if (s.group == 32) launch_norm<T, 32, 8>(backward, a, grid, stream);
  else if (s.group == 64 && s.per_thread == 8) launch_norm<T, 64, 8>(backward, a, grid, stream);
  else if (s.group == 64) launch_norm<T, 64, 16>(backward, a, grid, stream);
  else if (s.group == 256 && s.per_thread == 8) launch_norm<T, 256, 8>(backward, a, grid, stream);
  else if (s.group == 256) launch_norm<T, 256, 16>(backward, a, grid, stream);
  else launch_norm<T, 512, 16>(backward, a, grid, stream);
}

int check_norm(DisnCtx* ctx, const DisnLayerNorm* a) {
  const char* f = "disn_layer_norm";
  if (!a) return disn_fail(ctx, DISN_E_ARG, "%s: null arguments", f);
  if (!dense_type_ok(a->type) || a->reserved) return disn_fail(ctx, DISN_E_ARG, "%s: bad type %d or reserved field", f, a->type);
  if (!dense_size_ok(a->rows) || a->d < 1 || a->d > DISN_LAYER_NORM_MAX)
    return disn_fail(ctx, DISN_E_ARG, "%s: %lld rows of %lld (want d in 1..%d)", f, (long long)a->rows, (long long)a->d, DISN_LAYER_NORM_MAX);
  if (!(a->eps >= 0.0) || a->eps > 3e38) return disn_fail(ctx, DISN_E_ARG, "%s: eps must be a finite number >= 0", f);
  const size_t s = dense_type_size(a->type);
  if (!dense_matrix_ok(a->x, a->rows, a->d, a->ldx, s, true) || !dense_matrix_ok(a->y, a->rows, a->d, a->ldy, s, false))
    return disn_fail(ctx, DISN_E_ARG, "%s: x or y is null, misaligned or has a bad row distance", f);
  if (!dense_aligned(a->weight, s) || !dense_aligned(a->bias, s) || !dense_aligned(a->mean, 4) || !dense_aligned(a->rstd, 4))
    return disn_fail(ctx, DISN_E_ARG, "%s: a vector is misaligned", f);
  return DISN_OK;
}

int check_norm_grad(DisnCtx* ctx, const DisnLayerNormGrad* a) {
  const char* f = "disn_layer_norm_backward";
  if (!a) return disn_fail(ctx, DISN_E_ARG, "%s: null arguments", f);
  if (!dense_type_ok(a->type) || a->reserved) return disn_fail(ctx, DISN_E_ARG, "%s: bad type %d or reserved field", f, a->type);
  if (!dense_size_ok(a->rows) || a->d < 1 || a->d > DISN_LAYER_NORM_MAX)
    return disn_fail(ctx, DISN_E_ARG, "%s: %lld rows of %lld (want d in 1..%d)", f, (long long)a->rows, (long long)a->d, DISN_LAYER_NORM_MAX);
  const size_t s = dense_type_size(a->type);
  if (!dense_matrix_ok(a->x, a->rows, a->d, a->ldx, s, true) || !dense_matrix_ok(a->dy, a->rows, a->d, a->lddy, s, true) ||
      (a->dx && !dense_matrix_ok(a->dx, a->rows, a->d, a->lddx, s, false)) ||
      (a->residual && !dense_matrix_ok(a->residual, a->rows, a->d, a->ldr, s, true)))
    return disn_fail(ctx, DISN_E_ARG, "%s: a matrix is null, misaligned or has a bad row distance", f);
  if (a->rows && (!a->mean || !a->rstd)) return disn_fail(ctx, DISN_E_ARG, "%s: mean and rstd of the forward pass are needed", f);
  if (!dense_aligned(a->weight, s) || !dense_aligned(a->dweight, s) || !dense_aligned(a->dbias, s) || !dense_aligned(a->mean, 4) ||
      !dense_aligned(a->rstd, 4))
    return disn_fail(ctx, DISN_E_ARG, "%s: a vector is misaligned", f);
  return DISN_OK;
}

size_t norm_grad_workspace(const DisnLayerNormGrad* a) {
  if (!a->dweight && !a->dbias) return 0;
  const int64_t grid = norm_backward_grid(norm_shape(a->d), a->type, a->rows);
  return grid == 1 ? 0 : (size_t)grid * 2 * a->d * sizeof(float);
}

}  // namespace

extern "C" int disn_layer_norm(DisnCtx* ctx, const DisnLayerNorm* a, void* stream_) {
  if (!ctx) return DISN_E_ARG;
  DISN_TRY(check_norm(ctx, a));
  if (a->rows == 0) return DISN_OK;
  DISN_HIP(ctx, hipSetDevice(ctx->device));
  NormArgs k{};
  k.x = a->x, k.weight = a->weight, k.bias = a->bias, k.y = a->y, k.mean = a->mean, k.rstd = a->rstd;
  k.ldx = a->ldx, k.ldy = a->ldy, k.rows = a->rows, k.d = (int)a->d, k.eps = (float)a->eps;
  const NormShape s = norm_shape(a->d);
  const int64_t per = norm_rows_at_once(s), want = (a->rows + per - 1) / per, most = s.group == 512 ? 512 : 4096;
  dense_dispatch(a->type, [&](auto t) {
    launch_norm<decltype(t)>(s, false, k, want < most ? want : most, (hipStream_t)stream_);
    return 0;
  });
  DISN_HIP(ctx, hipGetLastError());
  return DISN_OK;
}

extern "C" int disn_layer_norm_backward_workspace(DisnCtx* ctx, const DisnLayerNormGrad* a, size_t* bytes) {
  if (!ctx) return DISN_E_ARG;
  if (!bytes) return disn_fail(ctx, DISN_E_ARG, "disn_layer_norm_backward_workspace: null result");
  DISN_TRY(check_norm_grad(ctx, a));
  *bytes = norm_grad_workspace(a);
  return DISN_OK;
}

extern "C" int disn_layer_norm_backward(DisnCtx* ctx, const DisnLayerNormGrad* a, void* workspace, size_t workspace_bytes,
                                        void* stream_) {
  if (!ctx) return DISN_E_ARG;
  DISN_TRY(check_norm_grad(ctx, a));
  if (!a->dx && !a->dweight && !a->dbias) return DISN_OK;
  const size_t need = norm_grad_workspace(a);
  if (need && (!workspace || !dense_aligned(workspace, 16) || workspace_bytes < need))
    return disn_fail(ctx, DISN_E_ARG, "disn_layer_norm_backward: needs %zu bytes of 16-byte aligned workspace", need);
  DISN_HIP(ctx, hipSetDevice(ctx->device));
  hipStream_t stream = (hipStream_t)stream_;
  NormArgs k{};
  k.x = a->x, k.dy = a->dy, k.mean_in = a->mean, k.rstd_in = a->rstd, k.weight = a->weight, k.residual = a->residual;
  k.y = a->dx, k.dweight = a->dweight, k.dbias = a->dbias, k.part = (float*)workspace;
  k.ldx = a->ldx, k.lddy = a->lddy, k.ldr = a->ldr, k.ldy = a->lddx, k.rows = a->rows, k.d = (int)a->d;
  const NormShape s = norm_shape(a->d);
  const int64_t grid = norm_backward_grid(s, a->type, a->rows);   // without rows one workgroup writes the empty sums
  dense_dispatch(a->type, [&](auto t) {
    using T = decltype(t);
    launch_norm<T>(s, true, k, grid, stream);
    if (need)
      k_sum_partials<T><<<(unsigned)((2 * a->d + 15) / 16), 256, 0, stream>>>(k.part, (int)grid, 2 * a->d, a->d, (T*)a->dweight,
                                                                              (T*)a->dbias);
    return 0;
  });
  DISN_HIP(ctx, hipGetLastError());
  return DISN_OK;
}
