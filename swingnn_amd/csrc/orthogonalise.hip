// Newton-Schulz orthogonalisation of update matrices, and the optimizer step that applies it.
//
//   X0 = G / (|G|_F + eps);   X <- a X + (b A + c A A) X  with  A = X X',  `steps` times
//
// with (a, b, c) = (3.4445, -4.7750, 2.0315).  Iteration, coefficients and the momentum below are those published as Muon
// (K. Jordan and others, 2024), the step's factor 0.2 sqrt(max(rows, cols)) is J. Liu and others' (2025).  The odd quintic
// pushes every singular value of X into [0.68, 1.21] and leaves the singular vectors, so the result is close to U V' of
// G = U S V'.  [0, 1.2024] is mapped into itself, so |X|_2 <= 1.2024, |A|_2 <= 1.45 and |B|_2 <= 2.81 (B = b A + c A A) from
// the first step on: fixed powers of two place X, A and B in fp16's range.  Matrices with more rows than columns are worked
// on as their transpose (m <= n throughout).
//
// Number formats.  The products run on fp16 MFMA with fp32 sums.  Rounding X itself is not an option: a step multiplies
// what lies in the weak directions by a = 3.44, rounding errors included (measured in 64 bits on rank-deficient G: 4e-2 of
// |O| with X in fp16, 0.3 in bf16).  X is therefore kept as a PAIR of fp16 numbers, X = hi + lo (22 bits, 4 bytes); the
// term a X uses both, the products read hi alone: their errors pass through B, whose left space is that of the strong
// directions, and are not multiplied up.  The diagonals of A and B, the largest entries, stay in fp32 vectors beside the
// fp16 off-diagonals.  Together, in an emulation of these roundings over nine shapes: 2e-4 ... 1.7e-3 of |O| for Gaussian,
// decaying and low-rank G, up to 2.8e-3 where all singular values are equal (bf16 operands: up to 1.5e-2).  A bf16 result
// is off by 1.7e-3 from its own rounding; with these it is 1.9e-3 ... 2.5e-3 on gradients, most where both sides are below 30.
//
// Every matrix of a call goes through the same launches: one for each 16 entries of the table (orthogonalise alone; the
// optimizer's table is kept), one to sum |G|^2 in parts (fp64), one to write X0, three per step (A, B, X; four where A's
// contraction is cut), one more in the optimizer where it clips.  A workgroup finds its matrix in a table of running tile
// counts (one load per lane and a ballot).  A and B are symmetric: the tiles on and below the diagonal are computed and
// written twice.  A call of small matrices alone takes one workgroup per matrix for all steps (k_orth_small).
//
// Measured, five steps, a call among others (fp32 G, a large library product in fp16 reaches 1107 TFLOP/s, a large copy
// 4.9 TB/s): 48 matrices of 384-channel blocks 445 ... 475 us, 2048 x 8192 (bf16 G) 805 ... 840 us = 680 TFLOP/s of the 558
// GFLOP that the symmetric halves need, 96 x 96 30 us.  Bounds, from the kernels' own times: A and B the stream from L2 into
// LDS (2048 x 8192, with the products taken out: 33 of 46 us remain of A, 21 of 24 of B); X at K = 2048 the same stream (66
// of 88 us); X at K = 384 neither rate: 47.5 us are 3.6 TB/s of its own reads and writes (hi, lo in; hi, lo out: 8 bytes an
// element; 4.1 TB/s of the measured bytes) and 340 TFLOP/s, with six stages between the two; below about 300 rows the
// launches, 4 to 10 us each.
#include "common.h"
#include <type_traits>

namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef __fp16 h4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) h4 lds_h4;
__device__ __forceinline__ f16x4 read_tr(const f16* p) {  // 4 rows x 16 columns per 16 lanes, delivered column per lane
  return __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_h4*)p));
}

constexpr float QA = 3.4445f, QB = -4.7750f, QC = 2.0315f;
constexpr float SX = 1024.f;     // X hi / lo hold X 2^10:  |X| <= 1.21  -> 1239
constexpr float SA = 8192.f;     // A holds A 2^13:         |A| <= 1.45  -> 11.9 k
constexpr float SB = 4096.f;     // B holds B 2^12:         |B| <= 2.81  -> 11.5 k

constexpr int NORM_ELEMS = 16384;  // elements per workgroup of the norm pass, at most NORM_PARTS of them per matrix
constexpr int NORM_PARTS = 1024;
constexpr int INIT_TILE = 64;

// one entry of a call: `batch` matrices of one shape (device copy in the plan, written by k_orth_table)
struct Item {
  const void* src;   // G: [batch][rows, cols], row stride ld_src, matrix stride bs_src (elements); NULL: momentum form
  void* dst;         // O, likewise
  int64_t ld_src, bs_src, ld_dst, bs_dst;
  int64_t off;       // byte offset of the first matrix's buffers in the workspace
  int64_t stride;    // bytes from one matrix's buffers to the next one's
  int64_t flat_off;  // momentum form: offset in the flat moment / EMA buffers
  int32_t rows, cols, m, n, mp, np, tall, batch;
  int32_t index;     // momentum form: place in the pointer tables
  int32_t parts;     // workgroups of the norm pass per matrix
  int64_t part_off;  // first fp64 partial of the item
  float scale;       // momentum form: update = lr scale O
  int32_t small;     // all steps in one workgroup
};
// running workgroup counts: norm, init, tiles of A, tiles of B, X product, whole small matrices, last X product
constexpr int PREFIXES = 7;
enum { P_NORM = 0, P_INIT, P_GRAM, P_POLY, P_FULL, P_SMALL, P_LAST };
struct Entry {
  Item item;
  int32_t end[PREFIXES];  // running totals including this item
};
constexpr int TABLE_BATCH = 16;
struct EntryBatch {
  Entry e[TABLE_BATCH];
};

__global__ void k_orth_table(EntryBatch b, int first, int count, int total, Item* __restrict__ items,
                             int32_t* __restrict__ ends) {
  const int i = threadIdx.x;
  if (i < count) {
    items[first + i] = b.e[i].item;
    for (int k = 0; k < PREFIXES; ++k) ends[k * total + first + i] = b.e[i].end[k];
  }
}

// Which item workgroup `bid` works on, and the first workgroup of that item: lane l looks at entry l
__device__ __forceinline__ int find_item(const int32_t* __restrict__ ends, int n, int bid, int& first) {
  first = 0;
  if (n == 1) return 0;
  const int lane = threadIdx.x & 63;
  for (int base = 0;; base += 64) {
    const int e = base + lane < n ? ends[base + lane] : 0x7fffffff;
    const unsigned long long before = __ballot(e <= bid);
    const int k = __popcll(before);
    if (k > 0) first = __builtin_amdgcn_readlane(e, k - 1);
    if (k < 64) return base + k;
  }
}

__device__ __forceinline__ int cdiv_up(int a, int b) { return (a + b - 1) / b; }

struct Bufs {
  char* x;
  size_t xbytes;
  f16 *lo, *A, *B;
  float *dA, *dB;
  __device__ __forceinline__ f16* hi(int k) const { return (f16*)(x + k * xbytes); }  // two of them, in turn
};
__device__ __forceinline__ Bufs bufs_of(const Item& I, char* ws, int b) {
  Bufs r;
  char* p = ws + I.off + (int64_t)b * I.stride;
  const size_t x = (size_t)I.mp * I.np * 2, a = (size_t)I.mp * I.mp * 2;
  r.x = p;
  r.xbytes = x;
  r.lo = (f16*)(p + 2 * x);
  r.A = (f16*)(p + 3 * x);
  r.B = (f16*)(p + 3 * x + a);
  r.dA = (float*)(p + 3 * x + 2 * a);
  r.dB = r.dA + I.mp;
  return r;
}

// momentum form (the optimizer step)
struct Momentum {
  const float* const* g_ptrs;
  float* const* p_ptrs;
  float* m;
  float* ema;
  int64_t total;
  const float* sqnorm;
  float max_norm, mu, lr, keep;  // keep = 1 - lr * weight_decay
  int32_t nesterov, n_ema;
  float ema_w[8];
  // the other parameters' chunks (for the clip's norm) and their partial sums
  const int32_t *numel, *chunk_tensor, *chunk_off;
  double* others;
  int32_t n_chunks, chunk;
};

__device__ __forceinline__ float clip_of(const Momentum& mo) {
  if (!mo.sqnorm) return 1.f;
  const float c = mo.max_norm / (sqrtf(*mo.sqnorm) + 1e-6f);
  return c > 1.f ? 1.f : c;  // a NaN norm stays NaN
}
__device__ __forceinline__ float new_m(const Momentum& mo, float m, float g) { return mo.mu * m + (1.f - mo.mu) * g; }
__device__ __forceinline__ float update_of(const Momentum& mo, float m_new, float g) {
  return mo.nesterov ? mo.mu * m_new + (1.f - mo.mu) * g : m_new;
}

// X lo is only ever read and written tile by tile: 16 x 32 tiles of 64 lanes x 8 elements, in the order of two
// neighbouring accumulators (lane l holds row l & 15, columns 4 (l >> 4) .. + 3 of the first and of the second)
__device__ __forceinline__ size_t lo_tile(int i, int j, int np) { return ((size_t)(i >> 4) * (np >> 5) + (j >> 5)) * 512; }
// Two neighbouring accumulators as packed fp16 (columns 4 lg .. of each) <-> 8 consecutive columns per lane, starting at
// 0, 16, 8, 24 for lane rows lg = 0 .. 3: swapping the odd lane rows of the first with the even ones of the second does
// both directions
__device__ __forceinline__ void swap_rows(f16x4& a, f16x4& b) {
  uint2 x = __builtin_bit_cast(uint2, a), y = __builtin_bit_cast(uint2, b);
  const auto p = __builtin_amdgcn_permlane16_swap(x.x, y.x, false, false);
  const auto q = __builtin_amdgcn_permlane16_swap(x.y, y.y, false, false);
  a = __builtin_bit_cast(f16x4, make_uint2(p[0], q[0]));
  b = __builtin_bit_cast(f16x4, make_uint2(p[1], q[1]));
}
__device__ __forceinline__ int swapped_col(int lg) { return 8 * (lg >> 1) + 16 * (lg & 1); }

// Where m and g nearly cancel, u is the rounding of its own fp32 sums and |u|^2 from the three sums the rounding of
// theirs; their quotient has no bound (1.5e6 in an emulation of 300 x 400), and above 1.2024 the quintic diverges.  |u|^2
// is therefore taken as at least 2^-34 of R^2 = (ca |m|)^2 + (cb |g|)^2.  u carries at most six roundings of either term,
// 6 2^-24 sqrt(2) R in all; fp64 sums of k terms in a chain move |u| by sqrt(k) 2^-26.5 sqrt(2) R: together below 0.2 of
// 2^-17 R for k < 4600 (up to 10^9 elements), so |X0| < 1.2.  Updates above 2^-17 R are what they were.
constexpr double CANCEL = 1.0 / (1ull << 34);

__device__ __forceinline__ double block_sum(double s, double* red) {  // 256 threads; all get the sum
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (red[0] + red[1]) + (red[2] + red[3]);
  __syncthreads();
  return s;
}

// Sums over a slice of a matrix into part[] (fp64: neither 1e-30 nor 1e30 leaves its range): |G|^2, or in the momentum form
// |g|^2, <g, m> and |m|^2.  The update u = a m + b c g is linear in the old m and in g, so these three give |u| for any clip
// factor c: the clip's norm and the updates' norms take one pass over g and m.  Workgroups behind the matrices' (momentum
// form) sum |g|^2 of the other parameters.
template <class T, bool MOM>
__global__ __launch_bounds__(256) void k_orth_norm(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                   int count, int blocks, double* __restrict__ part, Momentum mo) {
  __shared__ double red[4];
  constexpr int N = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  double s = 0.0, gm = 0.0, mm = 0.0;
  if (MOM && (int)blockIdx.x >= blocks) {
    const int wg = blockIdx.x - blocks, n_wg = gridDim.x - blocks;
    for (int c = wg; c < mo.n_chunks; c += n_wg) {
      const int t = mo.chunk_tensor[c], off = mo.chunk_off[c], n = min(mo.chunk, mo.numel[t] - off);
      const float* g = mo.g_ptrs[t] + off;
      for (int i = threadIdx.x; i < n; i += 256) s += (double)g[i] * (double)g[i];
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) mo.others[wg] = s;
    return;
  }
  int first;
  const int it = find_item(ends, count, blockIdx.x, first);
  const Item& I = items[it];
  const int w = blockIdx.x - first, b = w / I.parts, k = w - b * I.parts;
  const int64_t numel = (int64_t)I.rows * I.cols;
  const int64_t per = ((numel + I.parts - 1) / I.parts + N - 1) / N * N;
  const int64_t lo = k * per, hi = lo + per < numel ? lo + per : numel;
  if constexpr (MOM) {
    const float* g = mo.g_ptrs[I.index];
    const float* m = mo.m + I.flat_off;
    int64_t i = lo + threadIdx.x * N;
    auto add = [&](const vec& gv, const vec& mv) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const double a = gv[e], c = mv[e];
        s += a * a;
        gm += a * c;
        mm += c * c;
      }
    };
    constexpr int U = 4, W = 256 * N;  // U vectors of each in flight
    for (; i + (U - 1) * W + N <= hi; i += U * W) {
      vec gv[U], mv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        gv[u] = *reinterpret_cast<const vec*>(g + i + u * W);
        mv[u] = *reinterpret_cast<const vec*>(m + i + u * W);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) add(gv[u], mv[u]);
    }
    for (; i + N <= hi; i += W) add(*reinterpret_cast<const vec*>(g + i), *reinterpret_cast<const vec*>(m + i));
    for (; i < hi; ++i) {  // fewer than N left: one lane's
      const double a = g[i], c = m[i];
      s += a * a;
      gm += a * c;
      mm += c * c;
    }
  } else {
    const T* g = (const T*)I.src + (int64_t)b * I.bs_src;
    const bool flat = I.ld_src == I.cols;
    // rows one after the other where they are contiguous, else row by row
    const int64_t r_end = flat ? 1 : I.rows;
    for (int64_t r = flat ? 0 : k; r < r_end; r += I.parts) {
      const T* row = g + r * I.ld_src;
      const int64_t a = flat ? lo : 0, z = flat ? hi : I.cols;
      int64_t i = a + threadIdx.x * N;
      for (; i + N <= z; i += 256 * N) {
        const vec v = *reinterpret_cast<const vec*>(row + i);
#pragma unroll
        for (int e = 0; e < N; ++e) s += (double)(float)v[e] * (double)(float)v[e];
      }
      for (; i < z; ++i) s += (double)(float)row[i] * (double)(float)row[i];
    }
  }
  s = block_sum(s, red);
  double* out = part + (I.part_off + w) * (MOM ? 3 : 1);
  if constexpr (MOM) {
    gm = block_sum(gm, red);
    mm = block_sum(mm, red);
    if (threadIdx.x == 0) {
      out[1] = gm;
      out[2] = mm;
    }
  }
  if (threadIdx.x == 0) out[0] = s;
}

// |g|^2 of all parameters, in a fixed order
__global__ __launch_bounds__(256) void k_muon_sqnorm(const double* __restrict__ part, int n, const double* __restrict__ others,
                                                     int n_others, float* __restrict__ out) {
  __shared__ double red[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += part[3 * (size_t)i];
  for (int i = threadIdx.x; i < n_others; i += 256) s += others[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *out = (float)s;
}

// X0 = G / (|G|_F + eps) as hi + lo, transposed where the matrix is tall, zero in the padding.  One 64 x 64 tile of X: a wave
// writes 16 x 32 pairs of accumulator tiles as the products do.  Tall matrices come through LDS.
template <class T, bool MOM>
__global__ __launch_bounds__(256) void k_orth_init(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                   int count, const double* __restrict__ part, double eps,
                                                   char* __restrict__ ws, Momentum mo) {
  __shared__ double red[4];
  __shared__ float tile[INIT_TILE][INIT_TILE + 1];
  int first;
  const int it = find_item(ends, count, blockIdx.x, first);
  const Item& I = items[it];
  const int tm = cdiv_up(I.mp, INIT_TILE), tn = cdiv_up(I.np, INIT_TILE);
  int t = blockIdx.x - first;
  const int b = t / (tm * tn);
  t -= b * tm * tn;
  const int i0 = (t / tn) * INIT_TILE, j0 = (t % tn) * INIT_TILE;
  const Bufs B = bufs_of(I, ws, b);
  const T* g = MOM ? nullptr : (const T*)I.src + (int64_t)b * I.bs_src;
  const float* gm = MOM ? mo.g_ptrs[I.index] : nullptr;
  float* m = MOM ? mo.m + I.flat_off : nullptr;
  const float clip = MOM ? clip_of(mo) : 1.f;
  const int64_t ld = MOM ? I.cols : I.ld_src;
  // columns c .. c + 3 of row r of a matrix in G's layout, zero behind its edges
  auto four = [&](const auto* from, int r, int c, float (&v)[4]) {
    typedef std::remove_cv_t<std::remove_pointer_t<decltype(from)>> E;
    typedef E vec __attribute__((ext_vector_type(4), aligned(sizeof(E))));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = 0.f;
    if (r >= I.rows || c >= I.cols) return;
    const E* at = from + (int64_t)r * ld + c;
    if (c + 3 < I.cols) {
      const vec a = *reinterpret_cast<const vec*>(at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = (float)a[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < I.cols) v[e] = (float)at[e];
    }
  };
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, lg = lane >> 4;
  const bool tall = I.tall;
  const int ti = i0 + wave * 16;  // this wave's 16 rows of the tile, two pairs of column tiles
  // the four places of G that this thread reads: where they go in X, or 16 rows apart where the tile is transposed later
  float v[4][4], old[MOM ? 4 : 1][4];
  int gr[4], gc[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    gr[k] = tall ? j0 + k * 16 + (tid >> 4) : ti + l15;
    gc[k] = tall ? i0 + (tid & 15) * 4 : j0 + k * 16 + 4 * lg;
    if constexpr (MOM) {
      four(gm, gr[k], gc[k], v[k]);
      four((const float*)m, gr[k], gc[k], old[k]);
    } else {
      four(g, gr[k], gc[k], v[k]);
    }
  }
  if constexpr (MOM) {  // the tiles of X cover every element once: m moves on here
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      typedef float fvec __attribute__((ext_vector_type(4), aligned(4)));
      fvec o;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = v[k][e] * clip;
        o[e] = new_m(mo, old[k][e], a);
        v[k][e] = update_of(mo, o[e], a);
      }
      if (gr[k] >= I.rows || gc[k] >= I.cols) continue;
      float* at = m + (int64_t)gr[k] * ld + gc[k];
      if (gc[k] + 3 < I.cols) *reinterpret_cast<fvec*>(at) = o;
      else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (gc[k] + e < I.cols) at[e] = o[e];
      }
    }
  }
  if (tall) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[(tid & 15) * 4 + e][k * 16 + (tid >> 4)] = v[k][e];
  }
  const double* mine = part + (I.part_off + (int64_t)b * I.parts) * (MOM ? 3 : 1);
  double s = 0.0, gx = 0.0, mx = 0.0;
  for (int i = tid; i < I.parts; i += 256) {
    s += mine[i * (MOM ? 3 : 1)];
    if constexpr (MOM) {
      gx += mine[i * 3 + 1];
      mx += mine[i * 3 + 2];
    }
  }
  s = block_sum(s, red);
  if constexpr (MOM) {
    gx = block_sum(gx, red);
    mx = block_sum(mx, red);
    // u = ca m + cb g of the old m
    const double mu = mo.mu, ca = mo.nesterov ? mu * mu : mu, cb = (mo.nesterov ? (1.0 - mu) * (1.0 + mu) : 1.0 - mu) * clip;
    const double least = (ca * ca * mx + cb * cb * s) * CANCEL;
    s = ca * ca * mx + 2.0 * ca * cb * gx + cb * cb * s;
    s = s < least ? least : s;  // a NaN stays
  }
  const double inv = (double)SX / (sqrt(s) + eps);
  if (tall) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k][e] = tile[wave * 16 + l15][k * 16 + 4 * lg + e];
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int tj = j0 + q * 32;
    if (ti >= I.mp || tj >= I.np) continue;
    f16x4 h[2];
    f16x8 lv;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = (float)((double)v[2 * q + k][e] * inv);
        h[k][e] = (f16)x;
        lv[4 * k + e] = (f16)(x - (float)h[k][e]);
      }
    *reinterpret_cast<f16x8*>(B.lo + lo_tile(ti, tj, I.np) + lane * 8) = lv;
    swap_rows(h[0], h[1]);
    const f16x8 hv = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
    *reinterpret_cast<f16x8*>(B.hi(0) + (size_t)(ti + l15) * I.np + tj + swapped_col(lg)) = hv;
  }
}

template <int N>
__device__ __forceinline__ void wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
template <int PER, int NB>
__device__ __forceinline__ void wait_stage(int younger) {  // `younger` stages of PER transfers stay in flight
  if (NB >= 4 && younger >= 2) wait_vm<2 * PER>();
  else if (younger >= 1) wait_vm<PER>();
  else wait_vm<0>();
}

// place of column k of B inside its 32 columns: the MFMA slots of lane group g are k = 4 g .. 4 g + 3 and 16 + 4 g ..,
// the order in which the transposing LDS reads deliver X
__device__ __forceinline__ int b_perm(int k) { return (k & ~31) + 8 * ((k & 15) >> 2) + 4 * ((k >> 4) & 1) + (k & 3); }
// LDS rows of 64 contraction slots (8 chunks of 16 bytes): the chunk's place in row `row`, so that the fragment reads of 16
// rows spread over the banks.  LDS-DMA writes lanes in order, so the permutation is made on the global side.
__device__ __forceinline__ int nt_chunk(int row, int ch) { return ch ^ (row & 7); }

// A or B: T x T tile of a symmetric product P P' of one operand with contiguous contraction, T = 32 WT, 4 waves of
// 16 WT x 16 WT.  64-deep tiles of both row panels (whole 128-byte lines) go to LDS by LDS-DMA, NB stages.  What bounds it is
// the stream from L2 into LDS, about 14 TB/s: 32 flop per byte at T = 64 (460 TFLOP/s measured), 64 at T = 128.
// Whole calls of five steps, both sides in turn: tiles staged through registers two ahead instead of by LDS-DMA 222 against
// 169 us (1024^2), 924 against 846 us (2048 x 8192); both halves' fragments read before the products 175 against 170 and
// 860 against 852 us; eight stages where tiles are few 175 against 170 us (1024^2).
// PART / JOIN: few tiles of a long contraction.  PART: workgroup (slice, tile) writes its accumulators as they lie; JOIN adds
// a tile's slices in order and goes on as GRAM does.
enum { GRAM = 0, POLY, PART, JOIN };
constexpr int SYM_TILE = 64;
template <int KIND, int WT, int NB>
__global__ __launch_bounds__(256, 2) void k_orth_sym(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                     int count, int cur, int slices, float* __restrict__ parts,
                                                     char* __restrict__ ws) {
  constexpr int T = 32 * WT, OP = T * 64, STAGE = 2 * OP, PER = T / 32;
  __shared__ __attribute__((aligned(1024))) f16 sm[KIND == JOIN ? 8 : NB * STAGE];
  constexpr int IW = KIND == JOIN ? 1 : WT;  // JOIN: WT workgroups a tile, each with one row of every wave's accumulators
  const int tiles = KIND == PART ? gridDim.x / slices : gridDim.x / (KIND == JOIN ? WT : 1);
  const int wg = xcd_remap(blockIdx.x, gridDim.x), slice = KIND == PART ? wg / tiles : 0;
  const int bid = KIND == JOIN ? wg / WT : wg - slice * tiles, i_of = KIND == JOIN ? wg - bid * WT : 0;
  int first;
  const int it = find_item(ends, count, bid, first);
  const Item& I = items[it];
  const int mp = I.mp, nt = (mp + T - 1) / T, tpm = nt * (nt + 1) / 2;
  int t = bid - first;
  const int b = t / tpm;
  t -= b * tpm;
  int ti = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= t) ++ti;
  while (ti * (ti + 1) / 2 > t) --ti;
  const int tj = t - ti * (ti + 1) / 2;
  const Bufs B = bufs_of(I, ws, b);
  const f16* src = KIND == POLY ? B.A : B.hi(cur);
  const int ld = KIND == POLY ? mp : I.np;
  // this workgroup's share of the contraction, in 64-deep tiles
  const int nk_all = (ld + 63) / 64, k0 = KIND == PART ? (int)((int64_t)nk_all * slice / slices) : 0;
  const int k1 = KIND == PART ? (int)((int64_t)nk_all * (slice + 1) / slices) : nk_all;
  float* part = parts + ((size_t)slice * tiles + bid) * (T * T) + threadIdx.x * 4;
  const int p0 = ti * T, q0 = tj * T;
  const bool diag = ti == tj;  // both panels are the same one

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wp = wave >> 1, wq = wave & 1, l15 = lane & 15, lg = lane >> 4;
  f32x4 acc[IW][WT];
#pragma unroll
  for (int i = 0; i < IW; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  if constexpr (KIND != JOIN) {
    const f16 *gp[PER], *gq[PER];
    int gc[PER];
    unsigned dst[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = wave + 4 * i, row = 8 * j + (lane >> 3);
      gc[i] = nt_chunk(row, lane & 7) * 8;
      gp[i] = src + (size_t)min(p0 + row, mp - 1) * ld;
      gq[i] = src + (size_t)min(q0 + row, mp - 1) * ld;
      dst[i] = j * 1024;
    }
    const unsigned base = lds_addr(sm);
    auto issue = [&](int kt, int buf) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = min((k0 + kt) * 64 + gc[i], ld - 8);  // the last tile may be 32 deep: its second half is not multiplied
        lds_dma16(gp[i] + c, base + buf * (STAGE * 2) + dst[i]);
        if (!diag) lds_dma16(gq[i] + c, base + buf * (STAGE * 2) + OP * 2 + dst[i]);
      }
    };
    int fp[WT], fq[WT];
#pragma unroll
    for (int i = 0; i < WT; ++i) {  // rows 16 apart share their swizzle: 32 slots further is the chunk with bit 2 flipped
      const int rp = (wp * WT + i) * 16 + l15, rq = (wq * WT + i) * 16 + l15;
      fp[i] = rp * 64 + nt_chunk(rp, lg) * 8;
      fq[i] = (diag ? 0 : OP) + rq * 64 + nt_chunk(rq, lg) * 8;
    }
    const int nk = k1 - k0;
#pragma unroll
    for (int st = 0; st < NB - 1; ++st)
      if (st < nk) issue(st, st);
    int buf = 0;
    for (int kt = 0; kt < nk; ++kt) {
      if (diag) wait_stage<PER, NB>(min(nk - 1 - kt, NB - 2));
      else wait_stage<2 * PER, NB>(min(nk - 1 - kt, NB - 2));
      __syncthreads();
      if (kt + NB - 1 < nk) issue(kt + NB - 1, buf == 0 ? NB - 1 : buf - 1);
      const f16* s = sm + buf * STAGE;
      auto half = [&](int x) {
        f16x8 vp[WT], vq[WT];
#pragma unroll
        for (int i = 0; i < WT; ++i) {
          vp[i] = *reinterpret_cast<const f16x8*>(s + (fp[i] ^ x));
          vq[i] = *reinterpret_cast<const f16x8*>(s + (fq[i] ^ x));
        }
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
          for (int j = 0; j < WT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vp[i], vq[j], acc[i][j], 0, 0, 0);
      };
      half(0);
      if ((k0 + kt) * 64 + 32 < ld) half(32);
      buf = buf == NB - 1 ? 0 : buf + 1;
    }
  } else {
#pragma unroll 2
    for (int k = 0; k < slices; ++k)
#pragma unroll
      for (int j = 0; j < WT; ++j)
        acc[0][j] += *reinterpret_cast<const f32x4*>(part + (size_t)k * tiles * (T * T) + (i_of * WT + j) * 1024);
  }
  if constexpr (KIND == PART) {
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
      for (int j = 0; j < WT; ++j) *reinterpret_cast<f32x4*>(part + (i * WT + j) * 1024) = acc[i][j];
    return;
  }

  // lane: column q, rows p .. p + 3 of the product
#pragma unroll
  for (int j = 0; j < WT; ++j) {
    const int q = q0 + (wq * WT + j) * 16 + l15;
    if (q >= mp) continue;
    const float dq = KIND == POLY ? B.dA[q] : 0.f;
#pragma unroll
    for (int i = 0; i < IW; ++i) {
      const int p = p0 + (wp * WT + i + i_of) * 16 + 4 * lg;
      if (p >= mp) continue;
      f16x4 h;
      if constexpr (KIND != POLY) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          h[r] = (f16)(acc[i][j][r] * (SA / (SX * SX)));
          if (p + r == q) {
            B.dA[q] = acc[i][j][r] * (1.f / (SX * SX));
            h[r] = (f16)0.f;
          }
        }
        *reinterpret_cast<f16x4*>(B.A + (size_t)q * mp + p) = h;
        if (ti != tj) {
#pragma unroll
          for (int r = 0; r < 4; ++r) B.A[(size_t)(p + r) * mp + q] = h[r];
        }
      } else {
        const f16x4 o = *reinterpret_cast<const f16x4*>(B.A + (size_t)q * mp + p);
        const float4 dp = *reinterpret_cast<const float4*>(B.dA + p);
        const float dpv[4] = {dp.x, dp.y, dp.z, dp.w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float a = (float)o[r] * (1.f / SA), sq = acc[i][j][r] * (1.f / (SA * SA));
          h[r] = (f16)((QB * a + QC * (sq + (dpv[r] + dq) * a)) * SB);
          if (p + r == q) {
            B.dB[q] = QB * dq + QC * (sq + dq * dq);
            h[r] = (f16)0.f;
          }
        }
        *reinterpret_cast<f16x4*>(B.B + (size_t)q * mp + b_perm(p)) = h;
        if (ti != tj) {
          const int qp = b_perm(q);
#pragma unroll
          for (int r = 0; r < 4; ++r) B.B[(size_t)(p + r) * mp + qp] = h[r];
        }
      }
    }
  }
}

enum { MID = 0, OUT = 1, STEP = 2 };

// X' = a X + B X.  T x T tile, T = 32 WT.  B row-major (contiguous contraction), X [k][j] read through the transposing LDS
// read.  MID writes X' as hi + lo; OUT writes O in `otype`; STEP applies the optimizer's update and the moving averages.
template <int MODE, int WT, int NB>
__global__ __launch_bounds__(256, 2) void k_orth_apply(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                       int count, int cur, int otype, char* __restrict__ ws,
                                                       Momentum mo) {
  constexpr int T = 32 * WT, OP = T * 64, STAGE = 2 * OP, PER = T / 32;
  constexpr int XCH = T / 8;             // 16-byte chunks per X row in LDS
  constexpr int XROWS = 64 / XCH;        // X rows per wave transfer
  __shared__ __attribute__((aligned(1024))) f16 sm[NB * STAGE];
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
  int first;
  const int it = find_item(ends, count, bid, first);
  const Item& I = items[it];
  const int mp = I.mp, np = I.np, ntm = (mp + T - 1) / T, ntn = (np + T - 1) / T;
  int t = bid - first;
  const int b = t / (ntm * ntn);
  t -= b * ntm * ntn;
  const int i0 = (t % ntm) * T, j0 = (t / ntm) * T;
  const Bufs B = bufs_of(I, ws, b);
  const bool done = MODE == STEP && I.small;  // its steps are made: only the results are left to apply
  const f16* X = B.hi(done ? 0 : cur);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = wave >> 1, wj = wave & 1, l15 = lane & 15, lg = lane >> 4;
  const int q4 = l15 >> 2, p4 = l15 & 3;
  const f16 *gb[PER], *gx[PER];
  int gc[PER], gk[PER];
  unsigned dst[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = wave + 4 * i, row = 8 * j + (lane >> 3);
    gc[i] = nt_chunk(row, lane & 7) * 8;
    gb[i] = B.B + (size_t)min(i0 + row, mp - 1) * mp;
    gk[i] = XROWS * j + lane / XCH;
    const int sw = T == 128 ? 2 * (gk[i] & 7) : 2 * ((gk[i] >> 1) & 3);
    gx[i] = X + min(j0 + ((lane % XCH) ^ sw) * 8, np - 8);
    dst[i] = j * 1024;
  }
  const unsigned base = lds_addr(sm);
  auto issue = [&](int kt, int buf) {  // the last tile may be 32 deep: its second half is not multiplied
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      lds_dma16(gb[i] + min(kt * 64 + gc[i], mp - 8), base + buf * (STAGE * 2) + dst[i]);
      lds_dma16(gx[i] + (size_t)min(kt * 64 + gk[i], mp - 1) * np, base + buf * (STAGE * 2) + OP * 2 + dst[i]);
    }
  };
  int fb[WT], fx[WT];
  {
    const int r = 4 * lg + q4;  // the transposing read of k rows 4 lg .. and 16 + 4 lg ..: the swizzle is the same for both
    const int sw = T == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      const int rb = (wi * WT + i) * 16 + l15;
      fb[i] = rb * 64 + nt_chunk(rb, lg) * 8;
      const int lc = 2 * (wj * WT + i) + (p4 >> 1);
      fx[i] = OP + r * T + (lc ^ sw) * 8 + (p4 & 1) * 4;
    }
  }
  const int nk = done ? 0 : (mp + 63) / 64;
#pragma unroll
  for (int st = 0; st < NB - 1; ++st)
    if (st < nk) issue(st, st);
  // the accumulators start as (a X + diag(B) X) 2^22, read behind the first stages' transfers; in the result a lane holds
  // row i of X, columns j .. j + 3
  f32x4 acc[WT][WT];  // [i][j]
#pragma unroll
  for (int i = 0; i < WT; ++i) {
    const int ti = min(i0 + (wi * WT + i) * 16, mp - 16), ii = ti + l15;
    const float a = done ? 1.f : QA, e = done ? 0.f : B.dB[ii];
#pragma unroll
    for (int j = 0; j < WT; j += 2) {
      const int tj = min(j0 + (wj * WT + j) * 16, np - 32);
      const f16x8 hv = *reinterpret_cast<const f16x8*>(X + (size_t)ii * np + tj + swapped_col(lg));
      const f16x8 lv = *reinterpret_cast<const f16x8*>(B.lo + lo_tile(ti, tj, np) + lane * 8);
      f16x4 h[2] = {{hv[0], hv[1], hv[2], hv[3]}, {hv[4], hv[5], hv[6], hv[7]}};
      swap_rows(h[0], h[1]);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = (float)h[t][r];
          acc[i][j + t][r] = (a * (x + (float)lv[4 * t + r]) + e * x) * SB;
        }
    }
  }
  int buf = 0;
  for (int kt = 0; kt < nk; ++kt) {
    wait_stage<2 * PER, NB>(min(nk - 1 - kt, NB - 2));
    __syncthreads();
    if (kt + NB - 1 < nk) issue(kt + NB - 1, buf == 0 ? NB - 1 : buf - 1);
    const f16* s = sm + buf * STAGE;
    auto half = [&](int ks) {
      f16x8 vb[WT], vx[WT];
#pragma unroll
      for (int i = 0; i < WT; ++i) {
        vb[i] = *reinterpret_cast<const f16x8*>(s + (fb[i] ^ (32 * ks)));
        const f16x4 x0 = read_tr(s + fx[i] + 32 * T * ks), x1 = read_tr(s + fx[i] + (32 * ks + 16) * T);
        vx[i] = (f16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
      }
#pragma unroll
      for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vx[j], vb[i], acc[i][j], 0, 0, 0);
    };
    half(0);
    if (kt * 64 + 32 < mp) half(1);
    buf = buf == NB - 1 ? 0 : buf + 1;
  }

  if constexpr (MODE == MID) {
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      const int ti = i0 + (wi * WT + i) * 16;
#pragma unroll
      for (int j = 0; j < WT; j += 2) {
        const int tj = j0 + (wj * WT + j) * 16;  // mp and np are multiples of 32: a pair of tiles is in or out
        if (ti >= mp || tj >= np) continue;
        f16x4 h[2];
        f16x8 lv;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = acc[i][j + t][r] * (1.f / SB);
            h[t][r] = (f16)x;
            lv[4 * t + r] = (f16)(x - (float)h[t][r]);
          }
        *reinterpret_cast<f16x8*>(B.lo + lo_tile(ti, tj, np) + lane * 8) = lv;
        swap_rows(h[0], h[1]);
        const f16x8 hv = {h[0][0], h[0][1], h[0][2], h[0][3], h[1][0], h[1][1], h[1][2], h[1][3]};
        *reinterpret_cast<f16x8*>(B.hi(cur ^ 1) + (size_t)(ti + l15) * np + tj + swapped_col(lg)) = hv;
      }
    }
  }
  if constexpr (MODE != MID) {
    // through LDS in G's orientation, so that O (or the parameter and its averages) is touched in whole rows of the tile;
    // 32 WT = 128: the two halves of G's rows, which two of the waves hold each, one after the other
    constexpr int HR = T == 128 ? 64 : T, LD = T + 4;
    static_assert(HR * LD * 4 <= NB * STAGE * 2, "the tile reuses the stages");
    float* tile = reinterpret_cast<float*>(sm);
    const bool tall = I.tall;
    const int r0 = tall ? j0 : i0, c0 = tall ? i0 : j0;  // G's row and column of the tile
    float* p = nullptr;
    if constexpr (MODE == STEP) p = mo.p_ptrs[I.index];
    const float step = MODE == STEP ? mo.lr * I.scale : 0.f;
    for (int half = 0; half < T / HR; ++half) {
      __syncthreads();
      if (T == HR || (tall ? wj : wi) == half) {
#pragma unroll
        for (int i = 0; i < WT; ++i)
#pragma unroll
          for (int j = 0; j < WT; ++j) {
            const int li = (wi * WT + i) * 16 + l15, lj = (wj * WT + j) * 16 + 4 * lg;
            if (tall) {
#pragma unroll
              for (int r = 0; r < 4; ++r) tile[(lj + r - half * HR) * LD + li] = acc[i][j][r] * (1.f / (SB * SX));
            } else {
              *reinterpret_cast<f32x4*>(tile + (li - half * HR) * LD + lj) = acc[i][j] * (1.f / (SB * SX));
            }
          }
      }
      __syncthreads();
      if constexpr (MODE == OUT) {
#pragma unroll 2
        for (int k = tid; k < HR * (T / 8); k += 256) {
          const int lr = k / (T / 8), lc = (k % (T / 8)) * 8;
          const int gr = r0 + half * HR + lr, gc = c0 + lc;
          if (gr >= I.rows || gc >= I.cols) continue;
          const f32x4 x0 = *reinterpret_cast<const f32x4*>(tile + lr * LD + lc), x1 = *reinterpret_cast<const f32x4*>(tile + lr * LD + lc + 4);
          uint4 u;  // eight results of either type
          if (otype == SWG_BF16) {
            const uint2 a = pack_bf16x4(x0[0], x0[1], x0[2], x0[3]), c = pack_bf16x4(x1[0], x1[1], x1[2], x1[3]);
            u = make_uint4(a.x, a.y, c.x, c.y);
          } else {
            u = __builtin_bit_cast(uint4, (f16x8){(f16)x0[0], (f16)x0[1], (f16)x0[2], (f16)x0[3], (f16)x1[0], (f16)x1[1],
                                                  (f16)x1[2], (f16)x1[3]});
          }
          uint16_t* d = (uint16_t*)I.dst + (int64_t)b * I.bs_dst + (int64_t)gr * I.ld_dst + gc;
          typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2)));
          const vec w = __builtin_bit_cast(vec, u);
          if (gc + 7 < I.cols) *reinterpret_cast<vec*>(d) = w;
          else {
#pragma unroll
            for (int r = 0; r < 7; ++r)
              if (gc + r < I.cols) d[r] = w[r];
          }
        }
      } else {
#pragma unroll 1
        for (int k = tid; k < HR * (T / 4); k += 256) {
          const int lr = k / (T / 4), lc = (k % (T / 4)) * 4;
          const int gr = r0 + half * HR + lr, gc = c0 + lc;
          if (gr >= I.rows || gc >= I.cols) continue;
          const f32x4 x = *reinterpret_cast<const f32x4*>(tile + lr * LD + lc);
          const int have = min(4, I.cols - gc);
          const int64_t at = (int64_t)gr * I.cols + gc;
          float* pp = p + at;
          float* ee = mo.ema + I.flat_off + at;
          if (have == 4 && (((size_t)pp | (mo.n_ema ? (size_t)ee | (size_t)(mo.total * 4) : 0)) & 15) == 0) {
            f32x4 v = *reinterpret_cast<f32x4*>(pp), e[8];
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (q < mo.n_ema) e[q] = *reinterpret_cast<f32x4*>(ee + (int64_t)q * mo.total);
            v = mo.keep * v - step * x;
            *reinterpret_cast<f32x4*>(pp) = v;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (q < mo.n_ema) *reinterpret_cast<f32x4*>(ee + (int64_t)q * mo.total) = e[q] + mo.ema_w[q] * (v - e[q]);
          } else {
            for (int r = 0; r < have; ++r) {
              const float v = mo.keep * pp[r] - step * x[r];
              pp[r] = v;
              for (int q = 0; q < mo.n_ema; ++q) {
                float* e = ee + (int64_t)q * mo.total + r;
                *e += mo.ema_w[q] * (v - *e);
              }
            }
          }
        }
      }
    }
  }
}

// ---- small matrices: all steps in one workgroup ---------------------------------------------------------------------
// X stays in the accumulators of 8 waves for the whole call (fp32: no lo), its fp16 form in LDS; wave w owns the columns
// of tiles w njw .. of 16.  Per step: A by 32 x 32 blocks (K split over waves where there are few), B in A's place, then
// every wave multiplies its own columns and writes their fp16 form back (no other wave reads them before the barrier).
// Against 2 + 3 steps launches this saves their latencies, which are all that such a matrix costs there.  Measured, five
// steps, this form / the launches: 32 x 32 21 / 49 us, 96 x 96 32 / 65, 60 x 240 30 / 66, 96 x 384 47 / 77, 128 x 384 77 / 80,
// 32 x 2048 79 / 122, 512 of 96 x 96 66 / 180; a fourth column tile a wave at 128 rows spills (120 x 512: 112 / 86).
struct SmallGeom {
  int ldx, lda;  // row strides (elements) of X and A
  int off_a, off_d, off_red, bytes;
};
constexpr int SMALL_LDS = 163840, SMALL_WAVES = 8;
// number of waves that share the contraction of a 32 x 32 block of A
__host__ __device__ inline int small_split(int mp) { return mp == 32 ? 4 : mp == 64 ? 2 : 1; }
__host__ __device__ inline SmallGeom small_geom(int mp, int np) {
  SmallGeom g;
  g.ldx = np + 8;  // 16 bytes more than a multiple of the banks: the 16 rows of a fragment read spread over them
  g.lda = mp + 8;
  const int a = mp * g.lda * 2, nb = mp / 32, blocks = nb * (nb + 1) / 2;
  g.off_a = mp * g.ldx * 2;
  g.off_d = g.off_a + a;
  g.off_red = g.off_d + 2 * mp * 4;
  g.bytes = g.off_red + blocks * (small_split(mp) - 1) * 4096 + SMALL_WAVES * 8;
  return g;
}
__host__ __device__ inline int small_nj(int mt) { return mt == 2 ? 16 : mt == 4 ? 8 : mt == 6 ? 5 : 3; }  // column tiles a wave holds
inline bool is_small(int mp, int np) {
  return mp <= 128 && (np / 16 + SMALL_WAVES - 1) / SMALL_WAVES <= small_nj(mp / 16) && small_geom(mp, np).bytes <= SMALL_LDS;
}

// 0 that the compiler cannot see through: addresses formed with it are not kept in registers over the steps, where the
// accumulators need the room
__device__ __forceinline__ int opaque0() {
  int o;
  asm volatile("s_mov_b32 %0, 0" : "=s"(o));
  return o;
}

// X's row i, columns j .. j + 3, in a matrix of G's layout: a vector of four, or four rows where the matrix is tall
template <class T>
__device__ __forceinline__ f32x4 load4(const T* g, const Item& I, int64_t ld, bool tall, int i, int j) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (i >= I.m) return v;
  if (!tall && j + 3 < I.n) {
    const vec t = *reinterpret_cast<const vec*>(g + (int64_t)i * ld + j);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = (float)t[r];
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (j + r < I.n) v[r] = (float)g[tall ? (int64_t)(j + r) * ld + i : (int64_t)i * ld + j + r];
  }
  return v;
}
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));  // four rounded results of either type
template <class T, class V>
__device__ __forceinline__ void store4(T* g, const Item& I, int64_t ld, bool tall, int i, int j, V v) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (i >= I.m) return;
  if (!tall && j + 3 < I.n) {
    vec t;
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = (T)v[r];
    *reinterpret_cast<vec*>(g + (int64_t)i * ld + j) = t;
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (j + r < I.n) g[tall ? (int64_t)(j + r) * ld + i : (int64_t)i * ld + j + r] = (T)v[r];
  }
}

template <class T, bool MOM, int MT, int NJ>
__device__ __forceinline__ void small_body(const Item& I, int b, int steps, double eps, int otype, char* ws,
                                           char* lds) {
  const int m = I.m, mp = I.mp, np = I.np, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int l15 = lane & 15, lg = lane >> 4, q4 = l15 >> 2, p4 = l15 & 3;
  const SmallGeom G = small_geom(mp, np);
  f16* X = (f16*)lds;
  f16* A = (f16*)(lds + G.off_a);
  float *dA = (float*)(lds + G.off_d), *dB = dA + mp;
  double* red = (double*)(lds + G.off_red);
  float* scr = (float*)(lds + G.off_red);
  const int ntj = np / 16, njw = (ntj + SMALL_WAVES - 1) / SMALL_WAVES, jt0 = wave * njw;
  const bool tall = I.tall;
  constexpr int CH = 2;

  f32x4 x[MT][NJ];
  const Bufs W = MOM ? bufs_of(I, ws, b) : Bufs{};
  float inv = 1.f;
  int inv_exp = 0;  // 1 / (|G| + eps) as inv 2^inv_exp: it may lie outside fp32's range
  if constexpr (MOM) {  // X0 is there (the norm and the momentum take more bandwidth than one workgroup has)
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int jj = min(jt0 + j, ntj - 1) * 16;
        const f16x4 h = *reinterpret_cast<const f16x4*>(W.hi(0) + (size_t)(i * 16 + l15) * np + jj + 4 * lg);
        const f16x4 l = *reinterpret_cast<const f16x4*>(W.lo + lo_tile(i * 16, jj, np) + lane * 8 + (jj >> 4 & 1) * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][j][r] = (float)h[r] + (float)l[r];
      }
    }
  } else {
    double s = 0.0;
    const T* g = (const T*)I.src + (int64_t)b * I.bs_src;
    // up to CH tiles in flight at a time
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j0 = 0; j0 < NJ; j0 += CH) {
        __builtin_amdgcn_sched_barrier(0);
        const int ii = i * 16 + l15 + opaque0(), jb = (jt0 + j0) * 16 + 4 * lg, have = min(njw, ntj - jt0) - j0;
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          if (j0 + j >= NJ) continue;
          x[i][j0 + j] = (f32x4){0.f, 0.f, 0.f, 0.f};
          if (j < have) x[i][j0 + j] = load4(g, I, I.ld_src, tall, ii, jb + 16 * j);
        }
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          if (j0 + j >= NJ) continue;
#pragma unroll
          for (int r = 0; r < 4; ++r) s += (double)x[i][j0 + j][r] * (double)x[i][j0 + j][r];
        }
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int w = 0; w < SMALL_WAVES; ++w) s += red[w];
    inv = (float)frexp((double)SX / (sqrt(s) + eps), &inv_exp);
  }
  // this wave's columns of X as fp16: two neighbouring tiles would be 16 bytes a lane, one is 8
  auto put_hi = [&]() {
    const int o = opaque0();
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int ii = i * 16 + l15 + o;
        __builtin_amdgcn_sched_barrier(0);
        if (j >= njw || jt0 + j >= ntj) continue;
        *reinterpret_cast<f16x4*>(X + ii * G.ldx + (jt0 + j) * 16 + 4 * lg) =
            (f16x4){(f16)x[i][j][0], (f16)x[i][j][1], (f16)x[i][j][2], (f16)x[i][j][3]};
      }
  };
  if constexpr (!MOM) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][j][r] = ldexpf(x[i][j][r], inv_exp) * inv;
      }
  }
  put_hi();

  constexpr int NB2 = MT / 2, BLOCKS = NB2 * (NB2 + 1) / 2, S = MT == 2 ? 4 : MT == 4 ? 2 : 1;
  constexpr int ROUNDS = (BLOCKS * S + SMALL_WAVES - 1) / SMALL_WAVES;
  for (int step = 0; step < steps; ++step) {
    __syncthreads();  // X written
    f32x4 blk[ROUNDS][2][2];
    // unit u = (block, slice of the contraction): rows 32 bi .., columns 32 bj .. of A, bj <= bi
    auto unit = [&](int u, int& bi, int& bj, int& sl) {
      const int k = u % BLOCKS;
      sl = u / BLOCKS;
      bi = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3;
      bj = k - bi * (bi + 1) / 2;
    };
    auto product = [&](const f16* src, int ld, int bi, int bj, int k0, int k1, f32x4 (&c)[2][2]) {
      src += opaque0();
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q) c[p][q] = (f32x4){0.f, 0.f, 0.f, 0.f};
      const f16 *rp = src + (bi * 32 + l15) * ld + 8 * lg, *rq = src + (bj * 32 + l15) * ld + 8 * lg;
#pragma unroll 2
      for (int k = k0; k < k1; k += 32) {
        f16x8 vp[2], vq[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          vp[t] = *reinterpret_cast<const f16x8*>(rp + t * 16 * ld + k);
          vq[t] = *reinterpret_cast<const f16x8*>(rq + t * 16 * ld + k);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int q = 0; q < 2; ++q) c[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vp[p], vq[q], c[p][q], 0, 0, 0);
      }
    };
#pragma unroll
    for (int n = 0; n < ROUNDS; ++n) {
      const int u = wave + n * SMALL_WAVES;
      if (u >= BLOCKS * S) continue;
      int bi, bj, sl;
      unit(u, bi, bj, sl);
      const int nk = np / 32;
      product(X, G.ldx, bi, bj, nk * sl / S * 32, nk * (sl + 1) / S * 32, blk[n]);
      if (S > 1 && sl > 0) {
        float* to = scr + ((sl - 1) * BLOCKS + u % BLOCKS) * 1024 + lane * 4;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int q = 0; q < 2; ++q) *reinterpret_cast<f32x4*>(to + (p * 2 + q) * 256) = blk[n][p][q];
      }
    }
    if (S > 1) __syncthreads();
#pragma unroll
    for (int n = 0; n < ROUNDS; ++n) {
      const int u = wave + n * SMALL_WAVES;
      if (u >= BLOCKS) continue;  // slice 0
      int bi, bj, sl;
      unit(u, bi, bj, sl);
      const int oo = opaque0();
      if (S > 1) {
#pragma unroll
        for (int k = 1; k < S; ++k)
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              blk[n][p][q] += *reinterpret_cast<const f32x4*>(scr + ((k - 1) * BLOCKS + u) * 1024 + lane * 4 + (p * 2 + q) * 256);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int pp = oo + bi * 32 + p * 16 + 4 * lg, qq = bj * 32 + q * 16 + l15;
          f16x4 h;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = blk[n][p][q][r];
            h[r] = pp + r < m && qq < m && pp + r != qq ? (f16)(v * (SA / (SX * SX))) : (f16)0.f;
            if (pp + r == qq) dA[qq] = qq < m ? v * (1.f / (SX * SX)) : 0.f;
          }
          *reinterpret_cast<f16x4*>(A + qq * G.lda + pp) = h;
          if (bi != bj) {
#pragma unroll
            for (int r = 0; r < 4; ++r) A[(pp + r) * G.lda + qq] = h[r];
          }
        }
    }
    __syncthreads();  // A written
#pragma unroll
    for (int n = 0; n < ROUNDS; ++n) {
      const int u = wave + n * SMALL_WAVES;
      if (u >= BLOCKS) continue;
      int bi, bj, sl;
      unit(u, bi, bj, sl);
      const int oo = opaque0();
      product(A, G.lda, bi, bj, 0, mp, blk[n]);
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int pp = oo + bi * 32 + p * 16 + 4 * lg, qq = bj * 32 + q * 16 + l15;
          const f16x4 o = *reinterpret_cast<const f16x4*>(A + qq * G.lda + pp);
          const f32x4 dp = *reinterpret_cast<const f32x4*>(dA + pp);
          const float dq = dA[qq];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float a = (float)o[r] * (1.f / SA), sq = blk[n][p][q][r] * (1.f / (SA * SA));
            if (pp + r == qq) {
              dB[qq] = QB * dq + QC * (sq + dq * dq);
              blk[n][p][q][r] = 0.f;
            } else {
              blk[n][p][q][r] = (QB * a + QC * (sq + (dp[r] + dq) * a)) * SB;
            }
          }
        }
    }
    __syncthreads();  // A read
#pragma unroll
    for (int n = 0; n < ROUNDS; ++n) {
      const int u = wave + n * SMALL_WAVES;
      if (u >= BLOCKS) continue;
      int bi, bj, sl;
      unit(u, bi, bj, sl);
      const int oo = opaque0();
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int pp = oo + bi * 32 + p * 16 + 4 * lg, qq = bj * 32 + q * 16 + l15;
          const f32x4 v = blk[n][p][q];
          const f16x4 h = {(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
          *reinterpret_cast<f16x4*>(A + qq * G.lda + b_perm(pp)) = h;
          if (bi != bj) {
            const int qp = b_perm(qq);
#pragma unroll
            for (int r = 0; r < 4; ++r) A[(pp + r) * G.lda + qp] = h[r];
          }
        }
    }
    __syncthreads();  // B written
    const int o3 = opaque0();
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      const float e = dB[i * 16 + l15 + o3];
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[i][j][r] = (QA * x[i][j][r] + e * (float)(f16)x[i][j][r]) * SB;
    }
#pragma unroll
    for (int k = 0; k < MT / 2; ++k) {
      __builtin_amdgcn_sched_barrier(0);
      f16x8 vb[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) vb[i] = *reinterpret_cast<const f16x8*>(A + (i * 16 + l15 + o3) * G.lda + k * 32 + 8 * lg);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if (j >= njw || jt0 + j >= ntj) continue;
        const f16* at = X + (k * 32 + 4 * lg + q4 + o3) * G.ldx + (jt0 + j) * 16 + 4 * p4;
        const f16x4 x0 = read_tr(at), x1 = read_tr(at + 16 * G.ldx);
        const f16x8 vx = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
#pragma unroll
        for (int i = 0; i < MT; ++i) x[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vx, vb[i], x[i][j], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) x[i][j] *= 1.f / SB;
    if (step + 1 < steps) put_hi();
  }

#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (j >= njw || jt0 + j >= ntj) continue;
      __builtin_amdgcn_sched_barrier(0);
      const int ii = i * 16 + l15 + opaque0(), jj = (jt0 + j) * 16;
      if constexpr (MOM) {
        f16x4 h, l;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          h[r] = (f16)x[i][j][r];
          l[r] = (f16)(x[i][j][r] - (float)h[r]);
        }
        *reinterpret_cast<f16x4*>(W.hi(0) + (size_t)ii * np + jj + 4 * lg) = h;
        *reinterpret_cast<f16x4*>(W.lo + lo_tile(i * 16, jj, np) + lane * 8 + (jj >> 4 & 1) * 4) = l;
      } else {
        const f32x4 o = x[i][j] * (1.f / SX);
        const uint2 u = otype == SWG_BF16 ? pack_bf16x4(o[0], o[1], o[2], o[3])
                                          : __builtin_bit_cast(uint2, (f16x4){(f16)o[0], (f16)o[1], (f16)o[2], (f16)o[3]});
        store4((uint16_t*)I.dst + (int64_t)b * I.bs_dst, I, I.ld_dst, tall, ii, jj + 4 * lg, __builtin_bit_cast(u16x4, u));
      }
    }
}

template <class T, bool MOM>
__global__ __launch_bounds__(512, 1) void k_orth_small(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                       int count, int steps, double eps, int otype, char* __restrict__ ws) {
  extern __shared__ __attribute__((aligned(1024))) char dyn[];
  int first;
  const int it = find_item(ends, count, blockIdx.x, first);
  const Item& I = items[it];
  const int b = blockIdx.x - first;
  // by rows and by column tiles a wave holds: the fewer, the fewer registers
  const int njw = (I.np / 16 + SMALL_WAVES - 1) / SMALL_WAVES;
  switch (I.mp + (njw <= 2 ? 0 : njw <= 3 ? 1 : 2)) {
    case 32: small_body<T, MOM, 2, 2>(I, b, steps, eps, otype, ws, dyn); break;
    case 33: small_body<T, MOM, 2, 3>(I, b, steps, eps, otype, ws, dyn); break;
    case 34: small_body<T, MOM, 2, 16>(I, b, steps, eps, otype, ws, dyn); break;
    case 64: small_body<T, MOM, 4, 2>(I, b, steps, eps, otype, ws, dyn); break;
    case 65: small_body<T, MOM, 4, 3>(I, b, steps, eps, otype, ws, dyn); break;
    case 66: small_body<T, MOM, 4, 8>(I, b, steps, eps, otype, ws, dyn); break;
    case 96: small_body<T, MOM, 6, 2>(I, b, steps, eps, otype, ws, dyn); break;
    case 97: small_body<T, MOM, 6, 3>(I, b, steps, eps, otype, ws, dyn); break;
    case 98: small_body<T, MOM, 6, 5>(I, b, steps, eps, otype, ws, dyn); break;
    case 128: small_body<T, MOM, 8, 2>(I, b, steps, eps, otype, ws, dyn); break;
    default: small_body<T, MOM, 8, 3>(I, b, steps, eps, otype, ws, dyn); break;
  }
}

constexpr int OTHER_BLOCKS = 256;

// ---- host ----------------------------------------------------------------------------------------------------------
// What a call over a list of shapes needs; the same arithmetic sizes the workspace, fills the table and sizes the grids
struct Plan {
  int count = 0, wt_full = 2, wt_gram = 2;  // tile sides of the X product and of A, / 32
  int slices = 1;                           // of A's contraction
  int max_np = 0;
  int small_lds = 0;
  bool all_small = true, use_small = true;
  int64_t grid[PREFIXES] = {};
  int64_t parts = 0;
  size_t bytes = 0;                            // of X, A, B and the diagonals of all matrices
  double flops = 0;
};

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Small matrices take the one-workgroup form if the whole call does: beside larger ones the launches are there anyway, and
// more workgroups share the work.  Tile side of each product: 128 where that gives at least 1.5 workgroups a CU, else 64
bool plan_item(Plan& P, int32_t rows, int32_t cols, int32_t batch, bool mom, Item* I) {
  if (rows < 0 || cols < 0 || batch < 0 || rows > (1 << 20) || cols > (1 << 20)) return false;
  Item i = {};
  i.rows = rows; i.cols = cols; i.batch = batch;
  i.tall = rows > cols;
  i.m = i.tall ? cols : rows;
  i.n = i.tall ? rows : cols;
  i.mp = round_up(i.m, 32);
  i.np = round_up(i.n, 32);
  const int64_t numel = (int64_t)rows * cols;
  if (numel == 0) i.batch = 0;
  i.parts = (int)(cdiv64(numel, NORM_ELEMS) < NORM_PARTS ? cdiv64(numel, NORM_ELEMS) : NORM_PARTS);
  if (i.parts < 1) i.parts = 1;
  i.part_off = P.parts;
  i.off = (int64_t)P.bytes;
  if (i.batch && !is_small(i.mp, i.np)) P.all_small = false;
  i.small = P.use_small && is_small(i.mp, i.np);
  if (i.small) {
    const int lds = small_geom(i.mp, i.np).bytes;
    if (i.batch && lds > P.small_lds) P.small_lds = lds;
  }
  if (!i.small || mom) {
    i.stride = (int64_t)align256((size_t)3 * i.mp * i.np * 2 + (size_t)2 * i.mp * i.mp * 2 + (size_t)2 * i.mp * 4);
    P.parts += (int64_t)i.batch * i.parts;
  }
  P.bytes += (size_t)i.batch * (size_t)i.stride;
  P.flops += (double)i.batch * (3.0 * i.m * i.m * (double)i.n + (double)i.m * i.m * (double)i.m);
  P.count += 1;
  if (I) *I = i;
  return true;
}
void plan_grids(const Item& i, int wt_gram, int wt_full, bool mom, int64_t* g) {
  const int64_t nt = cdiv64(i.mp, SYM_TILE), ng = cdiv64(i.mp, 32 * wt_gram), b = i.batch, full = b * cdiv64(i.mp, 32 * wt_full) * cdiv64(i.np, 32 * wt_full);
  if (i.small) g[P_SMALL] += b;
  if (i.small && !mom) return;  // reads G and writes O by itself
  g[P_NORM] += b * i.parts;
  g[P_INIT] += b * cdiv64(i.mp, INIT_TILE) * cdiv64(i.np, INIT_TILE);
  g[P_LAST] += full;
  if (i.small) return;
  g[P_GRAM] += b * (ng * (ng + 1) / 2);
  g[P_POLY] += b * (nt * (nt + 1) / 2);
  g[P_FULL] += full;
}

// A of long matrices (a contraction of 2048 and more): 128-wide tiles where they are many, the contraction cut into slices of
// at least 512 until about 512 workgroups share the work.  Five steps, uncut / cut: 16 x 8192 302 / 97 us, 400 x 8192
// 429 / 190 us, 1024 x 4096 349 / 274 us, 2048 x 8192 (128-wide tiles) 961 / 875 us
void plan_slices(Plan& P) {  // grid[P_GRAM] holds 128-wide tiles
  P.wt_gram = 2;
  P.slices = 1;
  if (P.max_np < 2048 || P.grid[P_GRAM] == 0) return;
  int64_t tiles = P.grid[P_GRAM];
  if (tiles >= 100 && P.max_np >= 4096) P.wt_gram = 4;
  else tiles *= 4;  // about as many 64-wide ones
  const int64_t most = P.max_np / 512, want = 512 / tiles;
  P.slices = (int)(want < most ? want : most);
  if (P.slices <= 1) { P.slices = 1; P.wt_gram = 2; }
}

// plan buffer (device): Item[count], int32 ends[PREFIXES][count], then the fp64 partial sums
size_t table_bytes(int count) { return align256((size_t)count * sizeof(Item)) + align256((size_t)count * PREFIXES * 4); }

template <class F>
bool make_plan(int32_t count, bool mom, F shape, Plan& P) {  // shape(i, rows, cols, batch)
  if (count < 0) return false;
  for (int pass = 0; pass < 3; ++pass) {  // is every matrix small?  counts of 128-wide tiles, counts of the tiles chosen
    P.parts = 0; P.bytes = 0; P.flops = 0; P.count = 0; P.small_lds = 0; P.max_np = 0;
    for (int k = 0; k < PREFIXES; ++k) P.grid[k] = 0;
    for (int32_t i = 0; i < count; ++i) {
      int32_t r, c, b;
      shape(i, r, c, b);
      Item it;
      if (!plan_item(P, r, c, b, mom, &it)) return false;
      plan_grids(it, pass < 2 ? 4 : P.wt_gram, pass < 2 ? 4 : P.wt_full, mom, P.grid);
      if (it.batch && !it.small && it.np > P.max_np) P.max_np = it.np;
    }
    if (pass == 0) P.use_small = P.all_small;
    if (pass == 1) {
      P.wt_full = P.grid[P_LAST] >= 384 ? 4 : 2;
      plan_slices(P);
    }
  }
  for (int k = 0; k < PREFIXES; ++k)  // a launch holds fewer than 2^32 threads (the norm pass takes OTHER_BLOCKS more)
    if ((P.grid[k] + OTHER_BLOCKS) * (k == P_SMALL ? 512 : 256) > 0xffffffffll) return false;
  return true;
}

template <class F>
int write_table(int32_t count, const Plan& P, bool mom, F fill, void* table, hipStream_t s) {  // fill(i, item): the caller's fields
  Item* items = (Item*)table;
  int32_t* ends = (int32_t*)((char*)table + align256((size_t)count * sizeof(Item)));
  Plan run;
  run.use_small = P.use_small;
  int64_t g[PREFIXES] = {};
  for (int first = 0; first < count; first += TABLE_BATCH) {
    EntryBatch eb;
    const int n = count - first < TABLE_BATCH ? count - first : TABLE_BATCH;
    for (int k = 0; k < n; ++k) {
      fill(first + k, run, eb.e[k].item);
      plan_grids(eb.e[k].item, P.wt_gram, P.wt_full, mom, g);
      for (int q = 0; q < PREFIXES; ++q) eb.e[k].end[q] = (int32_t)g[q];
    }
    hipLaunchKernelGGL(k_orth_table, dim3(1), dim3(64), 0, s, eb, first, n, count, items, ends);
    SWG_LAUNCH_CHECK();
  }
  return 0;
}

struct Ptrs {
  const Item* items;
  const int32_t* ends;
  double* part;
  float* slices;
  char* ws;
  int count;
  const int32_t* end(int k) const { return ends + (size_t)k * count; }
};
size_t slice_bytes(const Plan& P) {  // partial tiles of A
  return P.slices == 1 ? 0 : (size_t)P.grid[P_GRAM] * P.slices * (size_t)(32 * P.wt_gram) * (32 * P.wt_gram) * 4;
}
size_t part_bytes(const Plan& P) { return align256(((size_t)P.parts * 3 + OTHER_BLOCKS) * 8); }
size_t ws_bytes_of(const Plan& P) { return part_bytes(P) + slice_bytes(P) + P.bytes; }
Ptrs ptrs_of(int count, const Plan& P, const void* table, void* ws) {
  Ptrs r;
  r.items = (const Item*)table;
  r.ends = (const int32_t*)((const char*)table + align256((size_t)count * sizeof(Item)));
  r.part = (double*)ws;
  r.slices = (float*)((char*)ws + part_bytes(P));
  r.ws = (char*)r.slices + slice_bytes(P);
  r.count = count;
  return r;
}

template <int KIND, int WT, int NB>
void sym(const Plan& P, const Ptrs& p, int g, int cur, hipStream_t s) {
  const int64_t per_tile = KIND == PART ? P.slices : KIND == JOIN ? WT : 1;
  hipLaunchKernelGGL((k_orth_sym<KIND, WT, NB>), dim3((unsigned)(P.grid[g] * per_tile)), dim3(256), 0, s, p.items, p.end(g),
                     p.count, cur, P.slices, p.slices, p.ws);
}
template <int MODE, int WT, int NB>
void apply(const Plan& P, const Ptrs& p, int cur, int otype, const Momentum& mo, hipStream_t s) {
  constexpr int G = MODE == MID ? P_FULL : P_LAST;
  hipLaunchKernelGGL((k_orth_apply<MODE, WT, NB>), dim3((unsigned)P.grid[G]), dim3(256), 0, s, p.items, p.end(G), p.count, cur,
                     otype, p.ws, mo);
}
// up to two workgroups a CU: three stages of each in flight in place of more workgroups.  Five steps of 1024 x 1024 (136
// tiles) 185 -> 170 us, of 251 x 1003 (10 tiles) 122 -> 113 us; 12 x 512 x 4096 keeps two stages, which are faster there
constexpr int64_t FEW_TILES = 512;
template <int MODE>
int run_steps(const Plan& P, const Ptrs& p, int steps, int otype, const Momentum& mo, hipStream_t s) {
  const bool only_last = P.grid[P_FULL] == 0;  // small matrices alone: their steps are made
  for (int k = only_last ? steps - 1 : 0, cur = 0; k < steps; ++k, cur ^= 1) {
    if (!only_last) {
      if (P.slices == 1 && P.grid[P_GRAM] <= FEW_TILES) sym<GRAM, 2, 4>(P, p, P_GRAM, cur, s);
      else if (P.slices == 1) sym<GRAM, 2, 2>(P, p, P_GRAM, cur, s);
      else if (P.wt_gram == 4) { sym<PART, 4, 2>(P, p, P_GRAM, cur, s); sym<JOIN, 4, 2>(P, p, P_GRAM, cur, s); }
      else { sym<PART, 2, 2>(P, p, P_GRAM, cur, s); sym<JOIN, 2, 2>(P, p, P_GRAM, cur, s); }
      if (P.grid[P_POLY] <= FEW_TILES) sym<POLY, 2, 4>(P, p, P_POLY, cur, s);
      else sym<POLY, 2, 2>(P, p, P_POLY, cur, s);
    }
    if (k + 1 < steps) {
      if (P.wt_full == 4) apply<MID, 4, 2>(P, p, cur, otype, mo, s);
      else apply<MID, 2, 3>(P, p, cur, otype, mo, s);
    } else {
      if (P.wt_full == 4) apply<MODE, 4, 2>(P, p, cur, otype, mo, s);
      else apply<MODE, 2, 3>(P, p, cur, otype, mo, s);
    }
    SWG_LAUNCH_CHECK();
  }
  return 0;
}

template <class T, bool MOM>
int run_all(const Plan& P, const Ptrs& p, int steps, int otype, float eps, const Momentum& mo, hipStream_t s,
            float* sqnorm = nullptr) {
  if (P.grid[P_NORM]) {
    const int blocks = (int)P.grid[P_NORM], extra = mo.n_chunks < OTHER_BLOCKS ? mo.n_chunks : OTHER_BLOCKS;
    hipLaunchKernelGGL((k_orth_norm<T, MOM>), dim3(blocks + extra), dim3(256), 0, s, p.items, p.end(P_NORM), p.count, blocks,
                       p.part, mo);
    if (MOM && mo.sqnorm)
      hipLaunchKernelGGL(k_muon_sqnorm, dim3(1), dim3(256), 0, s, p.part, blocks, mo.others, extra, sqnorm);
    hipLaunchKernelGGL((k_orth_init<T, MOM>), dim3((unsigned)P.grid[P_INIT]), dim3(256), 0, s, p.items, p.end(P_INIT), p.count,
                       p.part, (double)eps, p.ws, mo);
    SWG_LAUNCH_CHECK();
  }
  if (P.grid[P_SMALL]) {
    static std::atomic<uint64_t> ready{0};
    if (int e = ensure_dyn_lds(ready, (const void*)k_orth_small<T, MOM>, SMALL_LDS)) return e;
    hipLaunchKernelGGL((k_orth_small<T, MOM>), dim3((unsigned)P.grid[P_SMALL]), dim3(512), P.small_lds, s, p.items,
                       p.end(P_SMALL), p.count, steps, (double)eps, otype, p.ws);
    SWG_LAUNCH_CHECK();
  }
  return P.grid[P_LAST] ? run_steps<MOM ? STEP : OUT>(P, p, steps, otype, mo, s) : 0;
}

}  // namespace

extern "C" {

size_t swg_orthogonalise_workspace_bytes(int32_t count, const swg_orth_item* items) {
  if (count <= 0 || !items) return 0;
  Plan P;
  if (!make_plan(count, false, [&](int i, int32_t& r, int32_t& c, int32_t& b) { r = items[i].rows; c = items[i].cols; b = items[i].batch; }, P))
    return 0;
  return table_bytes(count) + ws_bytes_of(P) + 256;
}

int swg_orthogonalise(int32_t count, const swg_orth_item* items, int32_t itype, int32_t otype, int32_t steps, float eps,
                      void* ws, size_t ws_bytes, void* stream) {
  if (count < 0 || steps < 1 || steps > 64 || !(eps >= 0.f)) return SWG_E_SHAPE;
  if (count == 0) return 0;
  if (!items) return SWG_E_NULL;
  if (itype < SWG_F32 || itype > SWG_F16 || (otype != SWG_BF16 && otype != SWG_F16)) return SWG_E_UNSUPPORTED;
  Plan P;
  if (!make_plan(count, false, [&](int i, int32_t& r, int32_t& c, int32_t& b) { r = items[i].rows; c = items[i].cols; b = items[i].batch; }, P))
    return SWG_E_SHAPE;
  for (int i = 0; i < count; ++i) {
    const swg_orth_item& e = items[i];
    if (e.rows == 0 || e.cols == 0 || e.batch == 0) continue;
    if (!e.g || !e.out) return SWG_E_NULL;
    if (e.ld_g < e.cols || e.ld_out < e.cols) return SWG_E_SHAPE;
  }
  if (P.grid[P_LAST] + P.grid[P_SMALL] == 0) return 0;
  if (!ws) return SWG_E_NULL;
  if (ws_bytes < table_bytes(count) + ws_bytes_of(P) + 256) return SWG_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  void* table = (void*)(((size_t)ws + 255) & ~(size_t)255);
  SwgProfScope ps(KID_ORTH, P.flops * steps, 0.0, s);
  int r = write_table(count, P, false, [&](int i, Plan& run, Item& I) {
    const swg_orth_item& e = items[i];
    plan_item(run, e.rows, e.cols, e.batch, false, &I);
    I.src = e.g; I.dst = e.out; I.ld_src = e.ld_g; I.bs_src = e.bs_g; I.ld_dst = e.ld_out; I.bs_dst = e.bs_out;
  }, table, s);
  if (r) return r;
  const Ptrs p = ptrs_of(count, P, table, (char*)table + table_bytes(count));
  const Momentum none = {};
  if (itype == SWG_F32) return run_all<float, false>(P, p, steps, otype, eps, none, s);
  if (itype == SWG_BF16) return run_all<bf16, false>(P, p, steps, otype, eps, none, s);
  return run_all<f16, false>(P, p, steps, otype, eps, none, s);
}

static bool muon_plan(int32_t count, const swg_muon_item* items, Plan& P) {
  return make_plan(count, true, [&](int i, int32_t& r, int32_t& c, int32_t& b) { r = items[i].rows; c = items[i].cols; b = 1; }, P);
}

size_t swg_muon_table_bytes(int32_t count) { return count <= 0 ? 0 : table_bytes(count); }

size_t swg_muon_workspace_bytes(int32_t count, const swg_muon_item* items) {
  Plan P;
  if (count <= 0 || !items || !muon_plan(count, items, P)) return 0;
  return ws_bytes_of(P);
}

int swg_muon_table(int32_t count, const swg_muon_item* items, void* table, size_t table_size, void* stream) {
  if (count <= 0) return SWG_E_SHAPE;
  if (!items || !table) return SWG_E_NULL;
  Plan P;
  if (!muon_plan(count, items, P)) return SWG_E_SHAPE;
  for (int i = 0; i < count; ++i)
    if (items[i].rows < 1 || items[i].cols < 1 || items[i].flat_off < 0 || items[i].index < 0) return SWG_E_SHAPE;
  if (table_size < table_bytes(count) || ((size_t)table & 15)) return SWG_E_WORKSPACE;
  return write_table(count, P, true, [&](int i, Plan& run, Item& I) {
    plan_item(run, items[i].rows, items[i].cols, 1, true, &I);
    I.flat_off = items[i].flat_off; I.index = items[i].index; I.scale = items[i].scale;
  }, table, (hipStream_t)stream);
}

int swg_muon_ema_step(int32_t count, const swg_muon_item* items, const void* table, const void* p_ptrs, const void* g_ptrs,
                      float* m, float* ema, int64_t total, int32_t n_ema, const float* ema_decay, const int32_t* numel,
                      const int32_t* chunk_tensor, const int32_t* chunk_off, int32_t n_chunks, float* sqnorm, float max_norm,
                      float lr, float momentum, int32_t nesterov, float weight_decay, int32_t steps, float eps, void* ws,
                      size_t ws_bytes, void* stream) {
  if (count <= 0 || total <= 0 || n_ema < 0 || n_ema > 8 || steps < 1 || steps > 64 || n_chunks < 0 || !(eps >= 0.f))
    return SWG_E_SHAPE;
  if (!items || !table || !p_ptrs || !g_ptrs || !m || !ws || (n_ema > 0 && (!ema || !ema_decay))) return SWG_E_NULL;
  if (sqnorm && n_chunks > 0 && (!numel || !chunk_tensor || !chunk_off)) return SWG_E_NULL;
  Plan P;
  if (!muon_plan(count, items, P)) return SWG_E_SHAPE;
  if (ws_bytes < ws_bytes_of(P) || ((size_t)ws & 255) || ((size_t)table & 15)) return SWG_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const Ptrs p = ptrs_of(count, P, table, ws);
  Momentum mo = {};
  mo.g_ptrs = (const float* const*)g_ptrs; mo.p_ptrs = (float* const*)p_ptrs;
  mo.m = m; mo.ema = ema; mo.total = total; mo.sqnorm = sqnorm; mo.max_norm = max_norm; mo.mu = momentum; mo.lr = lr;
  mo.keep = 1.f - lr * weight_decay; mo.nesterov = nesterov; mo.n_ema = n_ema;
  for (int k = 0; k < n_ema; ++k) mo.ema_w[k] = 1.0f - ema_decay[k];
  if (sqnorm) {
    mo.numel = numel; mo.chunk_tensor = chunk_tensor; mo.chunk_off = chunk_off; mo.n_chunks = n_chunks;
    mo.chunk = swg_optim_chunk();
    mo.others = p.part + (size_t)P.parts * 3;
  }
  SwgProfScope ps(KID_ORTH, P.flops * steps, 0.0, s);
  return run_all<float, true>(P, p, steps, 0, eps, mo, s, sqnorm);
}

}  // extern "C"
