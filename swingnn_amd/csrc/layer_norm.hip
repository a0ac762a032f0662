// Layer norm over the last axis as an operator of its own, forward and backward, with the gradients of weight and bias
// reduced in a fixed order (no atomics: the same inputs give the same bits).
//
//   y  = (x - mean) r w + b,   r = 1 / sqrt(var + eps)          (mean, r kept in fp32 per row for the backward pass)
//   dx = r (g - mean(g) - xh mean(g xh)),   g = dy w,   xh = (x - mean) r
//   dw = sum_rows dy xh,   db = sum_rows dy
//
// Both passes are bound by HBM: x is read once and y written once; backward reads x and dy and writes dx.  A row is held
// in the registers of LANES lanes (8 .. 64: several rows per wavefront; 256 .. 1024: one row per workgroup) as V chunks
// of N elements (16 bytes), so mean and variance are two sums over registers: the mean's in 64 bits, the variance's of the
// centred values (no cancellation).  The backward pass reads the mean rounded to 32 bits.
// Loads carry the alignment of the ELEMENT only: gfx950 serves 16-byte loads at any address, so odd widths and row
// strides take the same path.  The last chunk of a width that N does not divide is moved back to end with the row: it
// overlaps its neighbour, whose columns it leaves out of the sums and stores a second time with the same values.
// Backward: lane and chunk fix the columns, so every lane sums dw / db of its columns over the rows of its workgroup in
// registers; the row groups of a workgroup are joined by shuffles and LDS, the workgroups by k_ln_cols.  The next row's
// x and dy are loaded before the present row's sums where the registers hold both.
// Measured (a large copy reaches 4.9 TB/s; kernel times under rocprofv3): forward 516096 x 96 fp32 76 us (5.2 TB/s; part of
// x stays in the memory-side cache), backward 184320 x 192 fp32 96 us (4.4 TB/s of x, dy, dx), 8192 x 4096 bf16 forward
// 25 us (5.4 TB/s), backward 50 us (4.0 TB/s, and 34 MB of partial sums), 4097 x 1001 fp16 forward 6.5, backward 15 + 4 us.
#include "common.h"
#include <type_traits>

namespace {

typedef _Float16 f16;

template <class T, int N>
struct Vec {
  typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T>
struct Vec<T, 1> {
  typedef T type __attribute__((ext_vector_type(1), aligned(sizeof(T))));
};

template <class T, int N>
__device__ __forceinline__ typename Vec<T, N>::type load_raw(const T* p) {
  return *reinterpret_cast<const typename Vec<T, N>::type*>(p);
}
template <class T, int N>
__device__ __forceinline__ void load_vec(const T* p, float* out) {
  const auto v = load_raw<T, N>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) out[e] = (float)v[e];
}
template <class T, int N>
__device__ __forceinline__ void store_vec(T* p, const float* in) {
  typename Vec<T, N>::type v;
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (T)in[e];
  *reinterpret_cast<typename Vec<T, N>::type*>(p) = v;
}

// Columns of chunk c of a row of D >= N elements: they start at `col`, the first `lo` of them belong to other chunks
// (lo = N: chunk c lies behind the row, its loads repeat the row's last chunk)
template <int N>
struct Cols {
  int col, lo;
  __device__ __forceinline__ Cols(int c, int D) {
    col = min(c * N, D - N);
    lo = min(c * N - col, N);
  }
};

__device__ __forceinline__ int cdiv_dev(int a, int b) { return (a + b - 1) / b; }

// group_sum() of common.h in 64 bits: both halves of the number move by the same register exchanges
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const uint2 u = __builtin_bit_cast(uint2, v);
  const uint2 o = make_uint2(__builtin_amdgcn_update_dpp(0u, u.x, CTRL, 0xf, 0xf, false),
                             __builtin_amdgcn_update_dpp(0u, u.y, CTRL, 0xf, 0xf, false));
  return v + __builtin_bit_cast(double, o);
}
template <int LANES>
__device__ __forceinline__ double group_sum64(double v) {
  if constexpr (LANES >= 16) {
    if constexpr (LANES == 64) {
      const uint2 u = __builtin_bit_cast(uint2, v);
      const auto x = __builtin_amdgcn_permlane32_swap(u.x, u.x, false, false), y = __builtin_amdgcn_permlane32_swap(u.y, u.y, false, false);
      v = __builtin_bit_cast(double, make_uint2(x[0], y[0])) + __builtin_bit_cast(double, make_uint2(x[1], y[1]));
    }
    if constexpr (LANES >= 32) {
      const uint2 u = __builtin_bit_cast(uint2, v);
      const auto x = __builtin_amdgcn_permlane16_swap(u.x, u.x, false, false), y = __builtin_amdgcn_permlane16_swap(u.y, u.y, false, false);
      v = __builtin_bit_cast(double, make_uint2(x[0], y[0])) + __builtin_bit_cast(double, make_uint2(x[1], y[1]));
    }
    v = dpp_add<0x128>(v);  // row_ror:8, 4, 2, 1
    v = dpp_add<0x124>(v);
    v = dpp_add<0x122>(v);
    v = dpp_add<0x121>(v);
  } else {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  }
  return v;
}

// Sum over the LANES lanes of a row.  LANES > 64: the whole workgroup; `red` alternates between two slots per call so
// that one barrier a call is enough.
template <int LANES, class A>
__device__ __forceinline__ A row_sum(A v, A* red, int& slot) {
  constexpr int G = LANES < 64 ? LANES : 64;
  if constexpr (sizeof(A) == 8) v = group_sum64<G>(v);
  else v = group_sum<G>(v);
  if constexpr (LANES <= 64) {
    return v;
  } else {
    constexpr int W = LANES / 64;
    A* r = red + slot * W;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    if constexpr (sizeof(A) == 8) {  // a 64-bit add takes longer: log2(W) of them in a chain, not W
      A t[W];
#pragma unroll
      for (int i = 0; i < W; ++i) t[i] = r[i];
#pragma unroll
      for (int n = W / 2; n > 0; n /= 2)
#pragma unroll
        for (int i = 0; i < n; ++i) t[i] += t[i + n];
      return t[0];
    }
    A s = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) s += r[i];
    return s;
  }
}

// The mean of a row from its sum in 64 bits, as a pair hi + lo: x - hi is exact for x near the mean, so x - hi - lo is as
// exact for a mean of 30000 as for one of 0.  A float32 sum leaves a few steps of the mean in every element, which
// r <= 1 / sqrt(eps) = 316 multiplies (rows of values around 30000.7, a few steps apart: y off by up to 3.3).  Sums of equal
// values are exact here (24 + 24 bits), and so is s - D hi.  `inv` is 1 / D.  Float32 / 64-bit sums: 516096 x 96 fp32
// 74.0 / 75.1 us, 184320 x 192 47.0 / 47.9 us, 8192 x 4096 bf16 24.1 / 24.9 us, 4096 x 16384 fp32 111.9 / 116.4 us.
// A chunk of a half type (11 bits at most) is summed in float32 first, which is exact for values within a factor of two.
template <class T, int N>
__device__ __forceinline__ double chunk_sum(const float* v, int lo) {  // of the elements from `lo` on
  typedef std::conditional_t<sizeof(T) == 2, float, double> A;
  A s = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) s += (A)(e >= lo ? v[e] : 0.f);
  return (double)s;
}
struct Mean {
  float hi, lo;
  __device__ __forceinline__ Mean(double s, int D, double inv) {
    hi = (float)(s * inv);
    lo = (float)((s - (double)D * (double)hi) * inv);
  }
};

template <int LANES>
constexpr int block_of() { return LANES <= 64 ? 256 : LANES; }

template <class T, class TW, int N, int LANES, int V>
__global__ __launch_bounds__(block_of<LANES>()) void k_ln_fwd(const T* __restrict__ x, int64_t ldx, int rows, int D,
                                                              const TW* __restrict__ w, const TW* __restrict__ b,
                                                              float eps, T* __restrict__ y, int64_t ldy,
                                                              float* __restrict__ mean_out,
                                                              float* __restrict__ rstd_out) {
  constexpr int BLK = block_of<LANES>(), RPB = BLK / LANES;
  __shared__ float red[2 * (LANES > 64 ? LANES / 64 : 1)];
  __shared__ double red_mean[2 * (LANES > 64 ? LANES / 64 : 1)];
  const int gl = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const bool ragged = D != N * LANES * V;
  const double inv = 1.0 / (double)D;
  int slot = 0;
  // the bound is the same for all lanes of a workgroup, so every barrier inside is reached by all of them
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < rows; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = min(row0 + grp, (int64_t)rows - 1);
    const bool live = row0 + grp < rows;
    const T* xr = x + row * ldx;
    float v[V][N];
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) load_vec<T, N>(xr + Cols<N>(gl + LANES * i, D).col, v[i]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (ragged) s += chunk_sum<T, N>(v[i], Cols<N>(gl + LANES * i, D).lo);
      else s += chunk_sum<T, N>(v[i], 0);
    }
    const Mean mean(row_sum<LANES>(s, red_mean, slot), D, inv);
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) v[i][e] = (v[i][e] - mean.hi) - mean.lo;
      if (ragged) {
        const int lo = Cols<N>(gl + LANES * i, D).lo;
#pragma unroll
        for (int e = 0; e < N; ++e) q += e >= lo ? v[i][e] * v[i][e] : 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) q += v[i][e] * v[i][e];
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<LANES>(q, red, slot) / (float)D + eps);
    if (live) {
      T* yr = y + row * ldy;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const Cols<N> c(gl + LANES * i, D);
        float ww[N], bb[N];
        if (w) load_vec<TW, N>(w + c.col, ww);
        if (b) load_vec<TW, N>(b + c.col, bb);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          float o = v[i][e] * rstd;
          if (w) o *= ww[e];
          if (b) o += bb[e];
          v[i][e] = o;
        }
        if (c.lo < N) store_vec<T, N>(yr + c.col, v[i]);
      }
      if (mean_out && gl == 0) {
        mean_out[row] = mean.hi;
        rstd_out[row] = rstd;
      }
    }
  }
}

// rows wider than the register forms: three walks over the row, the second and third out of L2
template <class T, class TW, int N>
__global__ __launch_bounds__(1024) void k_ln_fwd_wide(const T* __restrict__ x, int64_t ldx, int rows, int D,
                                                      const TW* __restrict__ w, const TW* __restrict__ b, float eps,
                                                      T* __restrict__ y, int64_t ldy, float* __restrict__ mean_out,
                                                      float* __restrict__ rstd_out) {
  __shared__ float red[32];
  __shared__ double red_mean[32];
  const int nch = cdiv_dev(D, N);
  const double inv = 1.0 / (double)D;
  int slot = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    double s = 0.0;
    float q = 0.f, v[N];
    for (int c = threadIdx.x; c < nch; c += 1024) {
      const Cols<N> cc(c, D);
      load_vec<T, N>(xr + cc.col, v);
      s += chunk_sum<T, N>(v, cc.lo);
    }
    const Mean mean(row_sum<1024>(s, red_mean, slot), D, inv);
    for (int c = threadIdx.x; c < nch; c += 1024) {
      const Cols<N> cc(c, D);
      load_vec<T, N>(xr + cc.col, v);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float c = (v[e] - mean.hi) - mean.lo;
        q += e >= cc.lo ? c * c : 0.f;
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<1024>(q, red, slot) / (float)D + eps);
    for (int c = threadIdx.x; c < nch; c += 1024) {
      const Cols<N> cc(c, D);
      float ww[N], bb[N];
      load_vec<T, N>(xr + cc.col, v);
      if (w) load_vec<TW, N>(w + cc.col, ww);
      if (b) load_vec<TW, N>(b + cc.col, bb);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[e] = ((v[e] - mean.hi) - mean.lo) * rstd;
        if (w) v[e] *= ww[e];
        if (b) v[e] += bb[e];
      }
      store_vec<T, N>(y + row * ldy + cc.col, v);
    }
    if (mean_out && threadIdx.x == 0) {
      mean_out[row] = mean.hi;
      rstd_out[row] = rstd;
    }
  }
}

// part: [gridDim.x][2][D] sums of dw and db over the rows of a workgroup, or NULL
template <class T, class TW, int N, int LANES, int V>
__global__ __launch_bounds__(block_of<LANES>()) void k_ln_bwd_rows(
    const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy, int64_t lddy, int rows, int D,
    const TW* __restrict__ w, const float* __restrict__ mean_in, const float* __restrict__ rstd_in, T* __restrict__ dx,
    int64_t lddx, float* __restrict__ part) {
  constexpr int BLK = block_of<LANES>(), RPB = BLK / LANES;
  constexpr bool AHEAD = V * N < 32 && BLK < 1024;  // both rows in registers; beyond that it spills
  extern __shared__ __attribute__((aligned(16))) float dyn[];  // [2][D] when LANES < BLK
  __shared__ float red[2 * (LANES > 64 ? LANES / 64 : 1)];
  const int gl = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const bool ragged = D != N * LANES * V;
  const float inv = 1.0f / (float)D;
  int slot = 0;
  float aw[V][N], ab[V][N];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) aw[i][e] = ab[i][e] = 0.f;
  typename Vec<T, N>::type rx[V], rg[V];
  float mean, rstd;
  const int64_t step = (int64_t)gridDim.x * RPB;
  auto fetch = [&](int64_t row0) {  // a group behind the last row repeats it, its values are masked below
    const int64_t row = min(row0 + grp, (int64_t)rows - 1);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int col = Cols<N>(gl + LANES * i, D).col;
      rx[i] = load_raw<T, N>(x + row * ldx + col);
      rg[i] = load_raw<T, N>(dy + row * lddy + col);
    }
    mean = mean_in[row];
    rstd = rstd_in[row];
  };
  if (AHEAD && (int64_t)blockIdx.x * RPB < rows) fetch((int64_t)blockIdx.x * RPB);
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < rows; row0 += step) {
    const int64_t row = row0 + grp;
    const bool live = row < rows;
    float xh[V][N], g[V][N];
    if (!AHEAD) fetch(row0);
    const float m = mean, r = rstd;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        xh[i][e] = ((float)rx[i][e] - m) * r;
        g[i][e] = (float)rg[i][e];
      }
    if (AHEAD && row0 + step < rows) fetch(row0 + step);
    if (ragged || row0 + RPB > rows) {
      // a select, not a product with 0: what is left out may be an infinity or NaN
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int lo = live ? Cols<N>(gl + LANES * i, D).lo : N;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float d = e >= lo ? g[i][e] : 0.f, h = e >= lo ? xh[i][e] : 0.f;
          aw[i][e] += d * h;
          ab[i][e] += d;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          aw[i][e] += g[i][e] * xh[i][e];
          ab[i][e] += g[i][e];
        }
    }
    if (!dx) continue;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const Cols<N> c(gl + LANES * i, D);
      if (w) {
        float ww[N];
        load_vec<TW, N>(w + c.col, ww);
#pragma unroll
        for (int e = 0; e < N; ++e) g[i][e] *= ww[e];
      }
      if (ragged) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          s1 += e >= c.lo ? g[i][e] : 0.f;
          s2 += e >= c.lo ? g[i][e] * xh[i][e] : 0.f;
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          s1 += g[i][e];
          s2 += g[i][e] * xh[i][e];
        }
      }
    }
    const float m1 = row_sum<LANES>(s1, red, slot) * inv, m2 = row_sum<LANES>(s2, red, slot) * inv;
    if (live) {
      T* dr = dx + row * lddx;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const Cols<N> c(gl + LANES * i, D);
#pragma unroll
        for (int e = 0; e < N; ++e) g[i][e] = r * (g[i][e] - m1 - xh[i][e] * m2);
        if (c.lo < N) store_vec<T, N>(dr + c.col, g[i]);
      }
    }
  }
  if (!part) return;
  if constexpr (LANES < 64) {  // row groups of a wavefront
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e)
#pragma unroll
        for (int o = LANES; o < 64; o <<= 1) {
          aw[i][e] += __shfl_xor(aw[i][e], o, 64);
          ab[i][e] += __shfl_xor(ab[i][e], o, 64);
        }
  }
  float* out = part + (size_t)blockIdx.x * 2 * D;
  if constexpr (LANES < BLK) {  // wavefronts of the workgroup, one after the other
    const int wave = threadIdx.x >> 6;
    for (int k = 0; k < BLK / 64; ++k) {
      if (wave == k && (int)(threadIdx.x & 63) < LANES) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const Cols<N> c(gl + LANES * i, D);
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (e >= c.lo) {
              dyn[c.col + e] = (k ? dyn[c.col + e] : 0.f) + aw[i][e];
              dyn[D + c.col + e] = (k ? dyn[D + c.col + e] : 0.f) + ab[i][e];
            }
        }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < 2 * D; c += BLK) out[c] = dyn[c];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const Cols<N> c(gl + LANES * i, D);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e >= c.lo) {
          out[c.col + e] = aw[i][e];
          out[D + c.col + e] = ab[i][e];
        }
    }
  }
}

// dx of rows wider than the register forms: two walks
template <class T, class TW, int N>
__global__ __launch_bounds__(1024) void k_ln_bwd_wide(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                      int64_t lddy, int rows, int D, const TW* __restrict__ w,
                                                      const float* __restrict__ mean_in,
                                                      const float* __restrict__ rstd_in, T* __restrict__ dx,
                                                      int64_t lddx) {
  __shared__ float red[32];
  const int nch = cdiv_dev(D, N);
  const float inv = 1.0f / (float)D;
  int slot = 0;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * ldx;
    const T* gr = dy + row * lddy;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float s1 = 0.f, s2 = 0.f, m1 = 0.f, m2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      for (int c = threadIdx.x; c < nch; c += 1024) {
        const Cols<N> cc(c, D);
        float xv[N], g[N], ww[N];
        load_vec<T, N>(xr + cc.col, xv);
        load_vec<T, N>(gr + cc.col, g);
        if (w) load_vec<TW, N>(w + cc.col, ww);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float xh = (xv[e] - mean) * rstd;
          if (w) g[e] *= ww[e];
          if (pass == 0) {
            s1 += e >= cc.lo ? g[e] : 0.f;
            s2 += e >= cc.lo ? g[e] * xh : 0.f;
          } else {
            g[e] = rstd * (g[e] - m1 - xh * m2);
          }
        }
        if (pass) store_vec<T, N>(dx + row * lddx + cc.col, g);
      }
      if (pass == 0) {
        m1 = row_sum<1024>(s1, red, slot) * inv;
        m2 = row_sum<1024>(s2, red, slot) * inv;
      }
    }
  }
}

// dw / db partial sums of rows wider than the register forms: a workgroup takes 256 columns of a slab of rows
template <class T>
__global__ __launch_bounds__(256) void k_ln_bwd_cols_wide(const T* __restrict__ x, int64_t ldx, const T* __restrict__ dy,
                                                          int64_t lddy, int rows, int D,
                                                          const float* __restrict__ mean_in,
                                                          const float* __restrict__ rstd_in, float* __restrict__ part) {
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= D) return;
  float aw = 0.f, ab = 0.f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float d = (float)dy[row * lddy + col];
    aw += d * (((float)x[row * ldx + col] - mean_in[row]) * rstd_in[row]);
    ab += d;
  }
  part[(size_t)blockIdx.y * 2 * D + col] = aw;
  part[(size_t)blockIdx.y * 2 * D + D + col] = ab;
}

// dw[col] / db[col] = sum over nblk partial rows, each thread a strided part, then 16 lanes through LDS in order
template <class TW>
__global__ __launch_bounds__(256) void k_ln_cols(const float* __restrict__ part, int nblk, int D, TW* __restrict__ dw,
                                                 TW* __restrict__ db) {
  __shared__ float red[16][17];
  const int c16 = threadIdx.x & 15, r16 = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c16;  // column of the [2 D] row
  float s = 0.f;
  if (col < 2 * D) {
    int r = r16;
    for (; r + 7 * 16 < nblk; r += 8 * 16) {
      float t[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) t[k] = part[(size_t)(r + 16 * k) * 2 * D + col];
#pragma unroll
      for (int k = 0; k < 8; ++k) s += t[k];
    }
    for (; r < nblk; r += 16) s += part[(size_t)r * 2 * D + col];
  }
  red[r16][c16] = s;
  __syncthreads();
  if (r16 == 0 && col < 2 * D) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[k][c16];
    if (col < D) {
      if (dw) dw[col] = (TW)t;
    } else if (db) {
      db[col - D] = (TW)t;
    }
  }
}

// Register form for `chunks` chunks of 16 bytes: -1 = none
// index: 0 (8,1) 1 (8,2) 2 (8,3) 3 (16,2) 4 (16,3) 5 (32,2) 6 (32,3) 7 (64,2) 8 (64,3) 9 (64,4) 10 (256,2) 11 (256,4)
//        12 (512,4) 13 (1024,4)
int ln_form(int chunks) {
  static const int cap[14] = {8, 16, 24, 32, 48, 64, 96, 128, 192, 256, 512, 1024, 2048, 4096};
  for (int i = 0; i < 14; ++i)
    if (chunks <= cap[i]) return i;
  return -1;
}
// Backward holds x, dy and two sums per column: 32 columns a lane fit 128 registers (1024 lanes) only for fp32's 16
int ln_form_bwd(int chunks, int elem_bytes) {
  const int form = ln_form(chunks);
  return form == 13 && elem_bytes == 2 ? -1 : form;
}
const int kLanes[14] = {8, 8, 8, 16, 16, 32, 32, 64, 64, 64, 256, 256, 512, 1024};

int bwd_blocks(int64_t rows, int D, int form) {
  if (rows <= 0) return 0;
  if (form < 0) return (int)(rows < 64 ? rows : 64);  // slabs of k_ln_bwd_cols_wide
  const int rpb = kLanes[form] <= 64 ? 256 / kLanes[form] : 1;
  const int64_t need = (rows + rpb - 1) / rpb;
  // two workgroups a CU.  Time of k_ln_bwd_rows in a sweep of its own (184320 x 192 fp32 / 8192 x 4096 bf16) with the next
  // row's loads in flight: 256 workgroups 91 / 51 us, 512: 84 / 45 us, 1024: 101 / 56 us; without them 1024 were best: 91 / 59 us
  return (int)(need < 512 ? need : 512);
}

// elements of a 16-byte chunk; widths below it go element by element
template <class T>
constexpr int chunk_n() { return 16 / (int)sizeof(T); }
static inline int chunks_of(int D, int n) { return D < n ? D : cdiv(D, n); }

template <class T, class TW>
int fwd(int64_t rows, int D, const T* x, int64_t ldx, const TW* w, const TW* b, float eps, T* y, int64_t ldy, float* mean,
        float* rstd, hipStream_t s) {
  constexpr int N = chunk_n<T>();
  const int form = ln_form(chunks_of(D, N));
  SwgProfScope ps(KID_LAYER_NORM, 0.0, 2.0 * rows * D * sizeof(T), s);
  if (form < 0) {
    hipLaunchKernelGGL((k_ln_fwd_wide<T, TW, N>), dim3((int)(rows < 4096 ? rows : 4096)), dim3(1024), 0, s, x, ldx, (int)rows, D,
                       w, b, eps, y, ldy, mean, rstd);
    SWG_LAUNCH_CHECK();
    return 0;
  }
  const int rpb = kLanes[form] <= 64 ? 256 / kLanes[form] : 1;
  const int64_t need = (rows + rpb - 1) / rpb;
  const int grid = (int)(need < 16384 ? need : 16384);
#define LNF(I, NN, LN, VV)                                                                                               \
  case I:                                                                                                            \
    hipLaunchKernelGGL((k_ln_fwd<T, TW, NN, LN, VV>), dim3(grid), dim3(block_of<LN>()), 0, s, x, ldx, (int)rows, D, w, b, eps, \
                       y, ldy, mean, rstd);                                                                          \
    break
  switch (D < N ? 100 : form) {
    LNF(100, 1, 8, 1);
    LNF(0, N, 8, 1); LNF(1, N, 8, 2); LNF(2, N, 8, 3); LNF(3, N, 16, 2); LNF(4, N, 16, 3); LNF(5, N, 32, 2); LNF(6, N, 32, 3);
    LNF(7, N, 64, 2); LNF(8, N, 64, 3); LNF(9, N, 64, 4); LNF(10, N, 256, 2); LNF(11, N, 256, 4); LNF(12, N, 512, 4); LNF(13, N, 1024, 4);
  }
#undef LNF
  SWG_LAUNCH_CHECK();
  return 0;
}

template <class T, class TW>
int bwd(int64_t rows, int D, const T* x, int64_t ldx, const T* dy, int64_t lddy, const TW* w, const float* mean,
        const float* rstd, T* dx, int64_t lddx, TW* dw, TW* db, float* part, hipStream_t s) {
  constexpr int N = chunk_n<T>();
  const int form = ln_form_bwd(chunks_of(D, N), (int)sizeof(T));
  const int nblk = bwd_blocks(rows, D, form);
  if (!dw && !db) part = nullptr;
  SwgProfScope ps(KID_LAYER_NORM, 0.0, (dx ? 3.0 : 2.0) * rows * D * sizeof(T), s);
  if (rows > 0) {
    if (form < 0) {
      if (dx) {
        hipLaunchKernelGGL((k_ln_bwd_wide<T, TW, N>), dim3((int)(rows < 4096 ? rows : 4096)), dim3(1024), 0, s, x, ldx, dy, lddy,
                           (int)rows, D, w, mean, rstd, dx, lddx);
        SWG_LAUNCH_CHECK();
      }
      if (part) {
        hipLaunchKernelGGL((k_ln_bwd_cols_wide<T>), dim3(cdiv(D, 256), nblk), dim3(256), 0, s, x, ldx, dy, lddy, (int)rows, D,
                           mean, rstd, part);
        SWG_LAUNCH_CHECK();
      }
    } else {
      const size_t lds = kLanes[form] <= 64 && part ? (size_t)2 * D * sizeof(float) : 0;  // <= 16 KiB
#define LNB(I, NN, LN, VV)                                                                                                 \
  case I:                                                                                                              \
    hipLaunchKernelGGL((k_ln_bwd_rows<T, TW, NN, LN, VV>), dim3(nblk), dim3(block_of<LN>()), lds, s, x, ldx, dy, lddy, (int)rows, \
                       D, w, mean, rstd, dx, lddx, part);                                                              \
    break
      switch (D < N ? 100 : form) {
        LNB(100, 1, 8, 1);
        LNB(0, N, 8, 1); LNB(1, N, 8, 2); LNB(2, N, 8, 3); LNB(3, N, 16, 2); LNB(4, N, 16, 3); LNB(5, N, 32, 2); LNB(6, N, 32, 3);
        LNB(7, N, 64, 2); LNB(8, N, 64, 3); LNB(9, N, 64, 4); LNB(10, N, 256, 2); LNB(11, N, 256, 4); LNB(12, N, 512, 4);
        case 13:
          if constexpr (sizeof(T) == 4)
            hipLaunchKernelGGL((k_ln_bwd_rows<T, TW, N, 1024, 4>), dim3(nblk), dim3(1024), 0, s, x, ldx, dy, lddy, (int)rows, D,
                               w, mean, rstd, dx, lddx, part);
      }
#undef LNB
      SWG_LAUNCH_CHECK();
    }
  }
  if (part || (rows == 0 && (dw || db))) {
    hipLaunchKernelGGL((k_ln_cols<TW>), dim3(cdiv(2 * D, 16)), dim3(256), 0, s, part, nblk, D, dw, db);
    SWG_LAUNCH_CHECK();
  }
  return 0;
}

int check_ln(int64_t rows, int D, int xt, int wt) {
  if (rows < 0 || rows > 0x7fffffff || D <= 0 || D > (1 << 24)) return SWG_E_SHAPE;
  if (xt < SWG_F32 || xt > SWG_F16 || !(wt == SWG_F32 || wt == xt)) return SWG_E_UNSUPPORTED;
  return 0;
}

// dispatch on (x type, weight type)
#define SWG_LN_TYPES(CALL)                                                   \
  do {                                                                       \
    if (xtype == SWG_F32) { typedef float T; typedef float TW; CALL; }        \
    if (xtype == SWG_BF16 && wtype == SWG_F32) { typedef bf16 T; typedef float TW; CALL; } \
    if (xtype == SWG_BF16) { typedef bf16 T; typedef bf16 TW; CALL; }         \
    if (wtype == SWG_F32) { typedef f16 T; typedef float TW; CALL; }          \
    { typedef f16 T; typedef f16 TW; CALL; }                                  \
  } while (0)

}  // namespace

extern "C" {

int swg_layer_norm_fwd(int64_t rows, int32_t D, const void* x, int64_t ldx, int32_t xtype, const void* w, const void* b,
                       int32_t wtype, float eps, void* y, int64_t ldy, float* mean, float* rstd, void* stream) {
  if (int r = check_ln(rows, D, xtype, wtype)) return r;
  if (rows == 0) return 0;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return SWG_E_NULL;
  if (ldx < 0 || ldy < D) return SWG_E_SHAPE;
  SWG_LN_TYPES(return (fwd<T, TW>(rows, D, (const T*)x, ldx, (const TW*)w, (const TW*)b, eps, (T*)y, ldy, mean, rstd,
                                  (hipStream_t)stream)));
}

size_t swg_layer_norm_bwd_workspace_bytes(int64_t rows, int32_t D, int32_t xtype) {
  if (check_ln(rows, D, xtype, xtype)) return 0;
  const int form = xtype == SWG_F32 ? ln_form_bwd(chunks_of(D, 4), 4) : ln_form_bwd(chunks_of(D, 8), 2);
  return align256((size_t)(bwd_blocks(rows, D, form) + 1) * 2 * D * sizeof(float));
}

int swg_layer_norm_bwd(int64_t rows, int32_t D, const void* x, int64_t ldx, const void* dy, int64_t lddy, int32_t xtype,
                       const void* w, int32_t wtype, const float* mean, const float* rstd, void* dx, int64_t lddx,
                       void* dw, void* db, void* ws, size_t ws_bytes, void* stream) {
  if (int r = check_ln(rows, D, xtype, wtype)) return r;
  if (rows > 0 && (!x || !dy || !mean || !rstd)) return SWG_E_NULL;
  if (ldx < 0 || lddy < 0 || (dx && lddx < D)) return SWG_E_SHAPE;
  if (dw || db) {
    if (!ws) return SWG_E_NULL;
    if (ws_bytes < swg_layer_norm_bwd_workspace_bytes(rows, D, xtype)) return SWG_E_WORKSPACE;
  }
  SWG_LN_TYPES(return (bwd<T, TW>(rows, D, (const T*)x, ldx, (const T*)dy, lddy, (const TW*)w, mean, rstd, (T*)dx, lddx,
                                  (TW*)dw, (TW*)db, (float*)ws, (hipStream_t)stream)));
}

}  // extern "C"
