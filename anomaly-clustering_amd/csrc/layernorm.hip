// Layer norm of rows, forward and backward (gfx950), for fp32, fp16 and bf16 rows of any width.
//
// forward   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
// backward  g = dy w, u = (x - mean) rstd:  dx = rstd (g - mean(g) - u mean(g u)),  dw = sum_rows dy u,  db = sum_rows dy
// Statistics, sums and gradients of the weights are fp32; the variance is taken from the differences (two passes over
// registers), and each result is rounded to its type once.
//
// Bound: memory.  A row lives in the registers of the wave or block that owns it, so x (and dy) are read once; a block of the
// backward pass walks over many rows with its share of dw and db in registers, and a second kernel adds the blocks' shares
// in a fixed order (no atomics: the same bits every time).  24571 x 4096 bf16: forward 86 us (4.7 TB/s), backward with its sums
// 117 us (5.2 TB/s); 25120 x 768 fp32: 25 and 40 us (a copy of that size stays in the cache: 6 .. 8 TB/s).  Widths that 16 bytes do not
// divide go entry by entry: 24571 x 1001 bf16 39 and 37 us (2.5, 4.0 TB/s), fp32 36 and 56 (5.4); over 16384 entries x is read in
// passes: 2000 x 32768 bf16 67 and 221 us.
#include <initializer_list>

#include "common.h"

namespace {

struct NormArgs {
  const void *x, *dy, *w, *b; void *y, *dx;
  int64_t x_row, dy_row, y_row, dx_row;          // strides in entries
  float *mean, *rstd; const float *mean_in, *rstd_in;
  float* part; int blocks;                       // backward: [blocks][2][C], dw then db
  void *dw, *db;
  int64_t rows; int C, w32; float eps;
};

template <class T, int VEC> struct Pack { typedef T type __attribute__((ext_vector_type(VEC))); };
template <class T> struct Pack<T, 1> { typedef T type; };
template <class T, int VEC>
__device__ inline void load(const T* p, float* v) {
  typename Pack<T, VEC>::type x = *reinterpret_cast<const typename Pack<T, VEC>::type*>(p);
  if constexpr (VEC == 1) v[0] = (float)x;
  else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (float)x[j];
  }
}
template <class T, int VEC>
__device__ inline void store(T* p, const float* v) {
  typename Pack<T, VEC>::type x;
  if constexpr (VEC == 1) x = (T)v[0];
  else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = (T)v[j];
  }
  *reinterpret_cast<typename Pack<T, VEC>::type*>(p) = x;
}
// VEC weights in the rows' type or fp32 (VEC of the rows: 16 bytes at most of theirs, 32 of fp32)
template <class T, int VEC>
__device__ inline void load_w(const void* p, int w32, int at, float* v) {
  if (w32) {
    constexpr int Q = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int j = 0; j < VEC; j += Q) load<float, Q>(static_cast<const float*>(p) + at + j, v + j);
  } else load<T, VEC>(static_cast<const T*>(p) + at, v);
}

// sums of two values over the L lanes of each of the W waves that share a row (L < 64: several rows to a wave)
template <int W, int L = 64>
__device__ inline void row_sum(float& a, float& b, float (*box)[2], int wave) {
  if constexpr (L == 64) {
    a = wave_sum(a);
    b = wave_sum(b);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) {
      a += __shfl_xor(a, o, 64);
      b += __shfl_xor(b, o, 64);
    }
  }
  if constexpr (W > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { box[wave][0] = a; box[wave][1] = b; }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) { a += box[i][0]; b += box[i][1]; }
  }
}

// N chunks of VEC entries per thread, W waves per row or L lanes (narrow rows); as many rows per block as its 256 threads hold.  One row per wave or block: a walk over
// several with the next one's loads ahead, as the backward pass does it, was slower (24571 x 4096 bf16: 86 us, 92 .. 100 walking).
// (five waves a SIMD at least: left to itself hipcc may fetch all weights at once into 210 registers - 8000 x 8192 fp32: 194 us, 101 so)
template <class T, int VEC, int N, int W, int L>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256, W > 4 ? 4 : 5) void norm_forward_kernel(const NormArgs a) {
  constexpr int R = W >= 4 ? 1 : 256 / L, THREADS = L * W;       // rows per block, threads per row
  typedef typename Pack<T, VEC>::type raw;
  __shared__ float box[W][2];
  const int tid = threadIdx.x, wave = tid >> 6, t = R == 1 ? tid : tid % THREADS;
  const int chunks = a.C / VEC;
  const int64_t row = (int64_t)blockIdx.x * R + (R == 1 ? 0 : tid / THREADS);
  if (row >= a.rows) return;                      // (all the lanes that a sum is taken over; R > 1 only with W == 1, where no barrier follows)
  {
    const T* from = static_cast<const T*>(a.x) + row * a.x_row;
    raw x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = t + THREADS * i;
      if (c < chunks) x[i] = *reinterpret_cast<const raw*>(from + c * VEC);
    }
    float v[N][VEC];
    float s = 0.f, zero = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (t + THREADS * i < chunks) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if constexpr (VEC == 1) v[i][j] = (float)x[i];
          else v[i][j] = (float)x[i][j];
          s += v[i][j];
        }
      }
    }
    row_sum<W, L>(s, zero, box, wave);
    const float mean = s / (float)a.C;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (t + THREADS * i < chunks) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { v[i][j] -= mean; q += v[i][j] * v[i][j]; }
      }
    }
    row_sum<W, L>(q, zero, box, wave);
    const float rstd = 1.0f / sqrtf(q / (float)a.C + a.eps);
    T* y = static_cast<T*>(a.y) + row * a.y_row;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = t + THREADS * i;
      if (c < chunks) {
        float w[VEC], b[VEC], o[VEC];
        if (a.w) load_w<T, VEC>(a.w, a.w32, c * VEC, w);
        if (a.b) load_w<T, VEC>(a.b, a.w32, c * VEC, b);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          o[j] = v[i][j] * rstd;
          if (a.w) o[j] *= w[j];
          if (a.b) o[j] += b[j];
        }
        store<T, VEC>(y + c * VEC, o);
      }
    }
    if (t == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
  }
}

// The next row's loads are issued before this row's sums are taken, so that a block always has two rows on their way (one row at
// a time: 133 us for 24571 x 4096 bf16, 4.5 TB/s).
template <class T, int VEC, int N, int W, int L>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void norm_backward_kernel(const NormArgs a) {
  constexpr int R = W >= 4 ? 1 : 256 / L, THREADS = L * W;       // rows in flight per block, threads per row
  typedef typename Pack<T, VEC>::type raw;
  __shared__ float box[W][2];
  __shared__ float share[R > 1 ? 2 * L * N * VEC : 1];
  const int tid = threadIdx.x, wave = tid >> 6, t = R == 1 ? tid : tid % THREADS, sub = R == 1 ? 0 : tid / THREADS;
  const int chunks = a.C / VEC;
  float w[N][VEC], dw[N][VEC], db[N][VEC];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = t + THREADS * i;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { w[i][j] = 1.f; dw[i][j] = db[i][j] = 0.f; }
    if (a.w && c < chunks) load_w<T, VEC>(a.w, a.w32, c * VEC, w[i]);
  }
  const float inv = 1.0f / (float)a.C;
  const int64_t step = (int64_t)gridDim.x * R;
  raw xr[N], gr[N];
  float mean = 0.f, rstd = 0.f;
  auto fetch = [&](int64_t row) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_row;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_row;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = t + THREADS * i;
      if (c < chunks) {
        xr[i] = *reinterpret_cast<const raw*>(x + c * VEC);
        gr[i] = *reinterpret_cast<const raw*>(dy + c * VEC);
      }
    }
    mean = a.mean_in[row];
    rstd = a.rstd_in[row];
  };
  int64_t row = (int64_t)blockIdx.x * R + sub;
  if (row < a.rows) fetch(row);
  for (; row < a.rows; row += step) {
    float u[N][VEC], g[N][VEC], s1 = 0.f, s2 = 0.f;
    const float r = rstd;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (t + THREADS * i < chunks) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          float xv, gv;
          if constexpr (VEC == 1) { xv = (float)xr[i]; gv = (float)gr[i]; } else { xv = (float)xr[i][j]; gv = (float)gr[i][j]; }
          u[i][j] = (xv - mean) * r;
          dw[i][j] += gv * u[i][j];
          db[i][j] += gv;
          g[i][j] = gv * w[i][j];
          s1 += g[i][j];
          s2 += g[i][j] * u[i][j];
        }
      }
    }
    if (row + step < a.rows) fetch(row + step);
    if (a.dx) {
      row_sum<W, L>(s1, s2, box, wave);
      s1 *= inv;
      s2 *= inv;
      T* dx = static_cast<T*>(a.dx) + row * a.dx_row;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = t + THREADS * i;
        if (c < chunks) {
          float o[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) o[j] = r * (g[i][j] - s1 - u[i][j] * s2);
          store<T, VEC>(dx + c * VEC, o);
        }
      }
    }
  }
  if (!a.part) return;
  if constexpr (R > 1) {                           // the block's rows one after the other, in their order
    for (int k = 0; k < R; ++k) {
      if (sub == k) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int at = (i * VEC + j) * L + t;
            share[at] = k ? share[at] + dw[i][j] : dw[i][j];
            share[L * N * VEC + at] = k ? share[L * N * VEC + at] + db[i][j] : db[i][j];
          }
      }
      __syncthreads();
    }
    if (sub) return;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        dw[i][j] = share[(i * VEC + j) * L + t];
        db[i][j] = share[L * N * VEC + (i * VEC + j) * L + t];
      }
  }
  float* p = a.part + (size_t)blockIdx.x * 2 * a.C;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = t + THREADS * i;
    if (c < chunks) {
      store<float, VEC < 4 ? VEC : 4>(p + c * VEC, dw[i]);
      store<float, VEC < 4 ? VEC : 4>(p + a.C + c * VEC, db[i]);
      if constexpr (VEC == 8) {
        store<float, 4>(p + c * VEC + 4, dw[i] + 4);
        store<float, 4>(p + a.C + c * VEC + 4, db[i] + 4);
      }
    }
  }
}

// Rows too wide for registers: one block per row, x read again for each pass (the second and third from a cache)
template <class T>
__global__ __launch_bounds__(1024) void norm_forward_wide_kernel(const NormArgs a) {
  __shared__ float box[16][2];
  const int wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_row;
  float s = 0.f, q = 0.f, zero = 0.f;
  for (int c = threadIdx.x; c < a.C; c += 1024) s += (float)x[c];
  row_sum<16>(s, zero, box, wave);
  const float mean = s / (float)a.C;
  for (int c = threadIdx.x; c < a.C; c += 1024) { const float d = (float)x[c] - mean; q += d * d; }
  row_sum<16>(q, zero, box, wave);
  const float rstd = 1.0f / sqrtf(q / (float)a.C + a.eps);
  T* y = static_cast<T*>(a.y) + row * a.y_row;
  for (int c = threadIdx.x; c < a.C; c += 1024) {
    float o = ((float)x[c] - mean) * rstd, w;
    if (a.w) { load_w<T, 1>(a.w, a.w32, c, &w); o *= w; }
    if (a.b) { load_w<T, 1>(a.b, a.w32, c, &w); o += w; }
    y[c] = (T)o;
  }
  if (threadIdx.x == 0 && a.mean) { a.mean[row] = mean; a.rstd[row] = rstd; }
}
template <class T>
__global__ __launch_bounds__(1024) void norm_backward_wide_kernel(const NormArgs a) {
  __shared__ float box[16][2];
  const int wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_row;
  const T* dy = static_cast<const T*>(a.dy) + row * a.dy_row;
  const float mean = a.mean_in[row], rstd = a.rstd_in[row];
  float s1 = 0.f, s2 = 0.f;
  for (int c = threadIdx.x; c < a.C; c += 1024) {
    float w = 1.f;
    if (a.w) load_w<T, 1>(a.w, a.w32, c, &w);
    const float g = (float)dy[c] * w;
    s1 += g;
    s2 += g * (((float)x[c] - mean) * rstd);
  }
  row_sum<16>(s1, s2, box, wave);
  s1 /= (float)a.C;
  s2 /= (float)a.C;
  T* dx = static_cast<T*>(a.dx) + row * a.dx_row;
  for (int c = threadIdx.x; c < a.C; c += 1024) {
    float w = 1.f;
    if (a.w) load_w<T, 1>(a.w, a.w32, c, &w);
    dx[c] = (T)(rstd * ((float)dy[c] * w - s1 - ((float)x[c] - mean) * rstd * s2));
  }
}
// ... and their columns: thread -> column, block row -> its share of the rows
template <class T>
__global__ __launch_bounds__(256) void norm_columns_kernel(const NormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = (float)(static_cast<const T*>(a.dy) + row * a.dy_row)[c];
    dw += g * (((float)(static_cast<const T*>(a.x) + row * a.x_row)[c] - a.mean_in[row]) * a.rstd_in[row]);
    db += g;
  }
  a.part[(size_t)blockIdx.y * 2 * a.C + c] = dw;
  a.part[(size_t)blockIdx.y * 2 * a.C + a.C + c] = db;
}

// Adds the blocks' shares: 32 columns x 32 groups of blocks per block, four shares in flight per thread (8 groups, one share at
// a time: 38 us for 1024 shares of 768 columns)
template <class T>
__global__ __launch_bounds__(1024) void norm_join_kernel(const NormArgs a) {
  __shared__ float sums[32][33];
  const int col = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + col;             // over 2 C: dw, then db
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < 2 * a.C) {
    const float* p = a.part + c;
    const size_t step = 2 * (size_t)a.C;
    int b = grp;
    for (; b + 96 < a.blocks; b += 128) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += p[(b + 32 * i) * step];
    }
    for (; b < a.blocks; b += 32) s[0] += p[b * step];
  }
  sums[grp][col] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (grp || c >= 2 * a.C) return;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 32; ++i) t[i & 3] += sums[i][col];
  const float sum = (t[0] + t[1]) + (t[2] + t[3]);
  void* out = c < a.C ? a.dw : a.db;
  const int at = c < a.C ? c : c - a.C;
  if (!out) return;
  if (a.w32) static_cast<float*>(out)[at] = sum;
  else static_cast<T*>(out)[at] = (T)sum;
}

// ---- which instance takes a width: VEC entries per access, N accesses per thread, W waves per row; N = 0: the wide kernels
struct Choice { int vec, n, w, l; };
Choice choose(int C, int size, bool aligned, int most) {         // most: entries of a row per thread
  Choice k;
  k.vec = aligned ? 16 / size : 1;
  const int64_t chunks = ((int64_t)C + k.vec - 1) / k.vec;
  k.l = 64;
  if (chunks <= 32) {                              // several rows to a wave (50000 x 192 bf16: forward 18 -> 12 us, backward 24 -> 19)
    k.n = k.w = 1;
    k.l = chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32;
    return k;
  }
  for (int w : {1, 4, 16}) {
    k.w = w;
    for (int n = 1; n <= most / k.vec; n *= 2) {
      k.n = n;
      if (chunks <= (int64_t)64 * w * n) return k;
    }
  }
  k.n = 0;
  return k;
}
// Blocks of the backward pass's row walk.  Each leaves a share of 8 C bytes, so twice the CUs where rows are long (100000 x 1000
// bf16: 114 us with 512 blocks, 134 with 1024; 24571 x 4096: 116 with 512, 131 with 256, 129 with 1024); narrow rows carry
// little, and more blocks keep more loads on their way (50000 x 192: 24 us with 1024, 27 with 512).
int backward_blocks(int64_t rows, int C, const Choice& k) {
  if (k.n == 0) return (int)max((int64_t)1, min((int64_t)64, rows));
  const int per = k.w >= 4 ? 1 : 256 / k.l;
  const int64_t most = k.w == 16 ? 256 : C <= 256 ? 1024 : 512;
  return (int)max((int64_t)1, min((rows + per - 1) / per, most));
}
// Entries of a row per thread: the backward pass holds five values for each, the forward pass one (20000 x 5120 fp16 forward: 97 us
// on four waves with 32, 148 on sixteen with 16; 24571 x 4096 bf16: 92 on four waves, 96 on one with 64)
constexpr int FORWARD = 32, BACKWARD = 16;

template <class T, int VEC, int N, int W, int L>
void launch_one(const NormArgs& a, bool backward, hipStream_t s) {
  constexpr int R = W >= 4 ? 1 : 256 / L, threads = W > 4 ? 64 * W : 256;
  if (backward) {
    if constexpr (N * VEC <= BACKWARD) hipLaunchKernelGGL((norm_backward_kernel<T, VEC, N, W, L>), dim3(a.blocks), dim3(threads), 0, s, a);
  } else hipLaunchKernelGGL((norm_forward_kernel<T, VEC, N, W, L>), dim3((unsigned)((a.rows + R - 1) / R)), dim3(threads), 0, s, a);
}
template <class T, int VEC, int N>
void launch_w(const NormArgs& a, const Choice& k, bool backward, hipStream_t s) {
  if constexpr (N == 1) {
    if (k.l == 8) return launch_one<T, VEC, 1, 1, 8>(a, backward, s);
    if (k.l == 16) return launch_one<T, VEC, 1, 1, 16>(a, backward, s);
    if (k.l == 32) return launch_one<T, VEC, 1, 1, 32>(a, backward, s);
  }
  if (k.w == 1) launch_one<T, VEC, N, 1, 64>(a, backward, s);
  else if (k.w == 4) launch_one<T, VEC, N, 4, 64>(a, backward, s);
  else launch_one<T, VEC, N, 16, 64>(a, backward, s);
}
template <class T, int VEC>
void launch_n(const NormArgs& a, const Choice& k, bool backward, hipStream_t s) {
  constexpr int most = (FORWARD > BACKWARD ? FORWARD : BACKWARD) / VEC;
  if (k.n == 1) return launch_w<T, VEC, 1>(a, k, backward, s);
  if constexpr (most >= 2) { if (k.n == 2) return launch_w<T, VEC, 2>(a, k, backward, s); }
  if constexpr (most >= 4) { if (k.n == 4) return launch_w<T, VEC, 4>(a, k, backward, s); }
  if constexpr (most >= 8) { if (k.n == 8) return launch_w<T, VEC, 8>(a, k, backward, s); }
  if constexpr (most >= 16) { if (k.n == 16) return launch_w<T, VEC, 16>(a, k, backward, s); }
  if constexpr (most >= 32) { if (k.n == 32) return launch_w<T, VEC, 32>(a, k, backward, s); }
}
// One thread block or part of one per row (the forward pass, the wide kernels' dx); a launch may not have 2^32 threads: 2^28 in each,
// one after the other
template <class T, class F>
void by_rows(const NormArgs& all, int threads, F launch_rows) {
  const int64_t most = (1LL << 28) / threads;
  for (int64_t r = 0; r < all.rows; r += most) {
    NormArgs a = all;
    a.rows = min(all.rows - r, most);
    a.x = static_cast<const T*>(all.x) + r * all.x_row;
    if (all.dy) a.dy = static_cast<const T*>(all.dy) + r * all.dy_row;
    if (all.y) a.y = static_cast<T*>(all.y) + r * all.y_row;
    if (all.dx) a.dx = static_cast<T*>(all.dx) + r * all.dx_row;
    if (all.mean) { a.mean = all.mean + r; a.rstd = all.rstd + r; }
    if (all.mean_in) { a.mean_in = all.mean_in + r; a.rstd_in = all.rstd_in + r; }
    launch_rows(a);
  }
}
template <class T>
void launch(const NormArgs& all, const Choice& k, bool backward, hipStream_t s) {
  if (k.n == 0) {
    if (!backward) by_rows<T>(all, 1024, [&](const NormArgs& a) { hipLaunchKernelGGL((norm_forward_wide_kernel<T>), dim3((unsigned)a.rows), dim3(1024), 0, s, a); });
    else {
      if (all.dx) by_rows<T>(all, 1024, [&](const NormArgs& a) { hipLaunchKernelGGL((norm_backward_wide_kernel<T>), dim3((unsigned)a.rows), dim3(1024), 0, s, a); });
      if (all.part) hipLaunchKernelGGL((norm_columns_kernel<T>), dim3((all.C + 255) / 256, all.blocks), dim3(256), 0, s, all);
    }
  } else {
    auto one = [&](const NormArgs& a) {
      if (k.vec == 1) launch_n<T, 1>(a, k, backward, s);
      else launch_n<T, 16 / (int)sizeof(T)>(a, k, backward, s);
    };
    if (backward) one(all);                        // its blocks walk over the rows
    else by_rows<T>(all, k.l * k.w, one);
  }
  if (backward && all.part) hipLaunchKernelGGL((norm_join_kernel<T>), dim3((2 * all.C + 31) / 32), dim3(1024), 0, s, all);
}

int check(const ac_norm_args* p, const char* what) {
  AC_REQUIRE(p, "%s: null arguments", what);
  AC_REQUIRE(p->type == AC_F32 || p->type == AC_F16 || p->type == AC_BF16, "%s: unknown type %d", what, p->type);
  AC_REQUIRE(p->weight_type == p->type || p->weight_type == AC_F32, "%s: weights must be fp32 or of the rows' type", what);
  AC_REQUIRE(p->rows >= 0 && p->rows < (1LL << 31), "%s: bad number of rows", what);
  AC_REQUIRE(p->width >= 1 && p->width <= 1 << 20, "%s: width %d must be in 1 .. 2^20", what, p->width);
  return AC_OK;
}
// 16-byte accesses where every address allows them
bool aligned16(const ac_norm_args* p, std::initializer_list<const void*> rows_of, std::initializer_list<int64_t> strides) {
  const int size = p->type == AC_F32 ? 4 : 2, vec = 16 / size;
  if (p->width % vec) return false;
  for (const void* q : rows_of) if ((uintptr_t)q & 15) return false;
  for (int64_t s : strides) if (s % vec) return false;
  return ((uintptr_t)p->weight & 15) == 0 && ((uintptr_t)p->bias & 15) == 0;
}

}  // namespace

extern "C" int ac_layer_norm(const ac_norm_args* p, void* stream) {
  if (int rc = check(p, "ac_layer_norm")) return rc;
  if (p->rows == 0) return AC_OK;
  AC_REQUIRE(p->x && p->y, "ac_layer_norm: null pointer");
  AC_REQUIRE(!p->mean == !p->rstd, "ac_layer_norm: mean and rstd come together");
  const int size = p->type == AC_F32 ? 4 : 2, wsize = p->weight_type == AC_F32 ? 4 : 2;
  AC_REQUIRE(((uintptr_t)p->x | (uintptr_t)p->y) % size == 0 && ((uintptr_t)p->weight | (uintptr_t)p->bias) % wsize == 0 &&
             (((uintptr_t)p->mean | (uintptr_t)p->rstd) & 3) == 0, "ac_layer_norm: misaligned pointer");
  NormArgs a = {};
  a.x = p->x; a.y = p->y; a.w = p->weight; a.b = p->bias; a.x_row = p->x_row; a.y_row = p->y_row;
  a.mean = p->mean; a.rstd = p->rstd; a.rows = p->rows; a.C = p->width; a.w32 = p->weight_type == AC_F32; a.eps = p->eps;
  const Choice k = choose(p->width, size, aligned16(p, {p->x, p->y}, {p->x_row, p->y_row}), FORWARD);
  if (p->type == AC_F32) launch<float>(a, k, false, as_stream(stream));
  else if (p->type == AC_F16) launch<_Float16>(a, k, false, as_stream(stream));
  else launch<__bf16>(a, k, false, as_stream(stream));
  return ac_check_launch("ac_layer_norm");
}

static int norm_shares(const ac_norm_args* p, bool aligned) {
  return backward_blocks(p->rows, p->width, choose(p->width, p->type == AC_F32 ? 4 : 2, aligned, BACKWARD));
}

// (a workspace for the one-entry kernels serves the 16-byte ones, and the other way round)
extern "C" size_t ac_layer_norm_backward_workspace_bytes(const ac_norm_args* p) {
  if (check(p, "ac_layer_norm_backward") != AC_OK || p->rows == 0 || (!p->dweight && !p->dbias)) return 0;
  return (size_t)max(norm_shares(p, true), norm_shares(p, false)) * 2 * p->width * sizeof(float);
}

extern "C" int ac_layer_norm_backward(const ac_norm_args* p, void* ws, size_t ws_bytes, void* stream) {
  if (int rc = check(p, "ac_layer_norm_backward")) return rc;
  const int size = p->type == AC_F32 ? 4 : 2, wsize = p->weight_type == AC_F32 ? 4 : 2;
  AC_REQUIRE(((uintptr_t)p->x | (uintptr_t)p->dy | (uintptr_t)p->dx) % size == 0 && (((uintptr_t)p->mean | (uintptr_t)p->rstd) & 3) == 0 &&
             ((uintptr_t)p->weight | (uintptr_t)p->dweight | (uintptr_t)p->dbias) % wsize == 0, "ac_layer_norm_backward: misaligned pointer");
  AC_REQUIRE(p->rows == 0 || (p->x && p->dy && p->mean && p->rstd), "ac_layer_norm_backward: null pointer");
  NormArgs a = {};
  a.x = p->x; a.dy = p->dy; a.dx = p->dx; a.w = p->weight; a.x_row = p->x_row; a.dy_row = p->dy_row; a.dx_row = p->dx_row;
  a.mean_in = p->mean; a.rstd_in = p->rstd; a.dw = p->dweight; a.db = p->dbias;
  a.rows = p->rows; a.C = p->width; a.w32 = p->weight_type == AC_F32;
  const size_t need = ac_layer_norm_backward_workspace_bytes(p);
  if (need && (!ws || ws_bytes < need)) return ac_fail(AC_EWORKSPACE, "ac_layer_norm_backward: workspace %zu < %zu", ws ? ws_bytes : (size_t)0, need);
  AC_REQUIRE(!need || ((uintptr_t)ws & 15) == 0, "ac_layer_norm_backward: the workspace must be 16-byte aligned");
  if (!p->dx && !p->dweight && !p->dbias) return AC_OK;
  const bool al = aligned16(p, {p->x, p->dy, p->dx}, {p->x_row, p->dy_row, p->dx_row});
  const Choice k = choose(p->width, size, al, BACKWARD);
  a.blocks = norm_shares(p, al);
  a.part = need ? static_cast<float*>(ws) : nullptr;
  if (p->rows == 0) {                              // nothing to walk over: the sums are zero
    a.blocks = 0;
    if (p->dweight || p->dbias) {
      if (p->type == AC_F32) hipLaunchKernelGGL((norm_join_kernel<float>), dim3((2 * a.C + 31) / 32), dim3(1024), 0, as_stream(stream), a);
      else if (p->type == AC_F16) hipLaunchKernelGGL((norm_join_kernel<_Float16>), dim3((2 * a.C + 31) / 32), dim3(1024), 0, as_stream(stream), a);
      else hipLaunchKernelGGL((norm_join_kernel<__bf16>), dim3((2 * a.C + 31) / 32), dim3(1024), 0, as_stream(stream), a);
    }
    return ac_check_launch("ac_layer_norm_backward");
  }
  if (p->type == AC_F32) launch<float>(a, k, true, as_stream(stream));
  else if (p->type == AC_F16) launch<_Float16>(a, k, true, as_stream(stream));
  else launch<__bf16>(a, k, true, as_stream(stream));
  return ac_check_launch("ac_layer_norm_backward");
}
