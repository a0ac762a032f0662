// Newton-Schulz orthogonalisation of update matrices, and the optimizer step that applies it.
//
//   X0 = G / (|G|_F + eps);   X <- a X + (b A + c A A) X  with  A = X X',  `steps` times
//
// with (a, b, c) = (3.4445, -4.7750, 2.0315): the odd quintic pushes every singular value of X into [0.68, 1.21] and
// leaves the singular vectors, so the result is close to U V' of G = U S V'.  [0, 1.2024] is mapped into itself, so
// |X|_2 <= 1.2024, |A|_2 <= 1.45 and |B|_2 <= 2.81 (B = b A + c A A) from the first step on: fixed powers of two place
// X, A and B in fp16's range.  Matrices with more rows than columns are worked on as their transpose (m <= n throughout).
//
// Number formats.  The products run on fp16 MFMA with fp32 sums.  Rounding X itself is not an option: a step multiplies
// what lies in the weak directions by a = 3.44, rounding errors included (measured in 64 bits on rank-deficient G: 4e-2 of
// |O| with X in fp16, 0.3 in bf16).  X is therefore kept as a PAIR of fp16 numbers, X = hi + lo (22 bits, 4 bytes); the
// term a X uses both, the products read hi alone: their errors pass through B, whose left space is that of the strong
// directions, and are not multiplied up.  The diagonals of A and B, the largest entries, stay in fp32 vectors beside the
// fp16 off-diagonals.  Together: 4e-5 ... 1.5e-3 of |O| for every spectrum tried (bf16 operands: up to 1.5e-2).
//
// Every matrix of a call goes through the same launches: one to sum |G|^2 in parts (fp64), one to write X0, three per
// step (A, B, X).  A workgroup finds its matrix in a table of running tile counts (one load per lane and a ballot).
// A and B are symmetric: the tiles on and below the diagonal are computed and written twice.
#include "common.h"

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
constexpr int NORM_PARTS = 256;
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
  int32_t pad_;
};
constexpr int PREFIXES = 5;  // running workgroup counts: norm, init, symmetric products, X product, (reserved)
enum { P_NORM = 0, P_INIT, P_SYM, P_FULL, P_SPARE };
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
  const int lane = threadIdx.x & 63;
  first = 0;
  for (int base = 0;; base += 64) {
    const int e = base + lane < n ? ends[base + lane] : 0x7fffffff;
    const unsigned long long before = __ballot(e <= bid);
    const int k = __popcll(before);
    if (k > 0) first = __builtin_amdgcn_readlane(e, k - 1);
    if (k < 64) return base + k;
  }
}

__device__ __forceinline__ int cdiv_up(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int xcd_remap(int bid, int nwg) {
  const int q = nwg >> 3, r = nwg & 7;
  const int xcd = bid & 7, slot = bid >> 3;
  return ((xcd < r) ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + slot;
}

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

// sum of squares of a slice of a matrix into part[] (fp64: neither 1e-30 nor 1e30 leaves its range).  Momentum form: also
// m <- mu m + (1 - mu) g, and the squares are the update's.
template <class T, bool MOM>
__global__ __launch_bounds__(256) void k_orth_norm(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                   int count, double* __restrict__ part, Momentum mo) {
  __shared__ double red[4];
  int first;
  const int it = find_item(ends, count, blockIdx.x, first);
  const Item& I = items[it];
  const int w = blockIdx.x - first, b = w / I.parts, k = w - b * I.parts;
  const int64_t numel = (int64_t)I.rows * I.cols;
  const int64_t per = ((numel + I.parts - 1) / I.parts + 3) & ~(int64_t)3;
  const int64_t lo = k * per, hi = lo + per < numel ? lo + per : numel;
  double s = 0.0;
  if constexpr (MOM) {
    const float* g = mo.g_ptrs[I.index];
    float* m = mo.m + I.flat_off;
    const float clip = clip_of(mo);
    for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
      const float gv = g[i] * clip, mv = new_m(mo, m[i], gv);
      m[i] = mv;
      const double u = update_of(mo, mv, gv);
      s += u * u;
    }
  } else {
    const T* g = (const T*)I.src + (int64_t)b * I.bs_src;
    const int cols = I.cols;
    if (I.ld_src == cols) {
      for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
        const double v = (double)(float)g[i];
        s += v * v;
      }
    } else {
      for (int64_t i = lo + threadIdx.x; i < hi; i += 256) {
        const int64_t r = i / cols;
        const double v = (double)(float)g[r * I.ld_src + (i - r * cols)];
        s += v * v;
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[I.part_off + w] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X0 = G / (|G|_F + eps) as hi + lo, transposed where the matrix is tall, zero in the padding.  One 64 x 64 tile of X.
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
  double s = (int)threadIdx.x < I.parts ? part[I.part_off + (int64_t)b * I.parts + threadIdx.x] : 0.0;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double inv = (double)SX / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + eps);
  const Bufs B = bufs_of(I, ws, b);
  const T* g = MOM ? nullptr : (const T*)I.src + (int64_t)b * I.bs_src;
  const float* gm = MOM ? mo.g_ptrs[I.index] : nullptr;
  const float* m = MOM ? mo.m + I.flat_off : nullptr;
  const float clip = MOM ? clip_of(mo) : 1.f;
  const int64_t ld = MOM ? I.cols : I.ld_src;
  auto value = [&](int r, int c) -> float {  // row and column of G
    if (r >= I.rows || c >= I.cols) return 0.f;
    const int64_t at = (int64_t)r * ld + c;
    float v;
    if constexpr (MOM) v = update_of(mo, m[at], gm[at] * clip);
    else v = (float)g[at];
    return (float)((double)v * inv);
  };
  if (I.tall) {
    for (int k = threadIdx.x; k < INIT_TILE * INIT_TILE; k += 256)
      tile[k & 63][k >> 6] = value(j0 + (k >> 6), i0 + (k & 63));
    __syncthreads();
  }
  for (int k = threadIdx.x; k < INIT_TILE * INIT_TILE; k += 256) {
    const int i = i0 + (k >> 6), j = j0 + (k & 63);
    if (i >= I.mp || j >= I.np) continue;
    const float v = I.tall ? tile[k >> 6][k & 63] : value(i, j);
    const f16 h = (f16)v;
    const size_t at = (size_t)i * I.np + j;
    B.hi(0)[at] = h;
    B.lo[at] = (f16)(v - (float)h);
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
__device__ __forceinline__ int nt_chunk(int row, int ch) { return ch ^ ((-(row >> 2)) & 3); }

// A (GRAM) or B (!GRAM): T x T tile of a symmetric product P P' of one operand with contiguous contraction, T = 32 WT,
// 4 waves of 16 WT x 16 WT.  32-deep tiles of both row panels go to LDS by LDS-DMA, NB stages.
template <bool GRAM, int WT, int NB>
__global__ __launch_bounds__(256, 2) void k_orth_sym(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                     int count, int cur, char* __restrict__ ws) {
  constexpr int T = 32 * WT, OP = T * 32, STAGE = 2 * OP, PER = T / 64;
  __shared__ __attribute__((aligned(1024))) f16 sm[NB * STAGE];
  const int bid = xcd_remap(blockIdx.x, gridDim.x);
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
  const f16* src = GRAM ? B.hi(cur) : B.A;
  const int ld = GRAM ? I.np : mp, K = ld;
  const int p0 = ti * T, q0 = tj * T;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wp = wave >> 1, wq = wave & 1, l15 = lane & 15, lg = lane >> 4;
  const f16 *gp[PER], *gq[PER];
  unsigned dst[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = wave + 4 * i, row = 16 * j + (lane >> 2), ch = nt_chunk(row, lane & 3) * 8;
    gp[i] = src + (size_t)min(p0 + row, mp - 1) * ld + ch;
    gq[i] = src + (size_t)min(q0 + row, mp - 1) * ld + ch;
    dst[i] = j * 1024;
  }
  const unsigned base = lds_addr(sm);
  auto issue = [&](int kt, int buf) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      lds_dma16(gp[i] + kt * 32, base + buf * (STAGE * 2) + dst[i]);
      lds_dma16(gq[i] + kt * 32, base + buf * (STAGE * 2) + OP * 2 + dst[i]);
    }
  };
  f32x4 acc[WT][WT];
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  int fp[WT], fq[WT];
#pragma unroll
  for (int i = 0; i < WT; ++i) {
    const int rp = (wp * WT + i) * 16 + l15, rq = (wq * WT + i) * 16 + l15;
    fp[i] = rp * 32 + nt_chunk(rp, lg) * 8;
    fq[i] = OP + rq * 32 + nt_chunk(rq, lg) * 8;
  }
  const int nk = K / 32;
#pragma unroll
  for (int st = 0; st < NB - 1; ++st)
    if (st < nk) issue(st, st);
  int buf = 0;
  for (int kt = 0; kt < nk; ++kt) {
    wait_stage<2 * PER, NB>(min(nk - 1 - kt, NB - 2));
    __syncthreads();
    if (kt + NB - 1 < nk) issue(kt + NB - 1, buf == 0 ? NB - 1 : buf - 1);
    const f16* s = sm + buf * STAGE;
    f16x8 vp[WT], vq[WT];
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      vp[i] = *reinterpret_cast<const f16x8*>(s + fp[i]);
      vq[i] = *reinterpret_cast<const f16x8*>(s + fq[i]);
    }
#pragma unroll
    for (int i = 0; i < WT; ++i)
#pragma unroll
      for (int j = 0; j < WT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vp[i], vq[j], acc[i][j], 0, 0, 0);
    buf = buf == NB - 1 ? 0 : buf + 1;
  }

  // lane: column q, rows p .. p + 3 of the product
#pragma unroll
  for (int j = 0; j < WT; ++j) {
    const int q = q0 + (wq * WT + j) * 16 + l15;
    if (q >= mp) continue;
    const float dq = GRAM ? 0.f : B.dA[q];
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      const int p = p0 + (wp * WT + i) * 16 + 4 * lg;
      if (p >= mp) continue;
      f16x4 h;
      if constexpr (GRAM) {
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
// The accumulator's four registers run along j (X's rows are G's rows) or, for tall matrices in OUT / STEP, along i.
template <int MODE, int WT, int NB>
__global__ __launch_bounds__(256, 2) void k_orth_apply(const Item* __restrict__ items, const int32_t* __restrict__ ends,
                                                       int count, int cur, int otype, char* __restrict__ ws,
                                                       Momentum mo) {
  constexpr int T = 32 * WT, OP = T * 32, STAGE = 2 * OP, PER = T / 64;
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
  const f16* X = B.hi(cur);

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = wave >> 1, wj = wave & 1, l15 = lane & 15, lg = lane >> 4;
  const int q4 = l15 >> 2, p4 = l15 & 3;
  const f16 *gb[PER], *gx[PER];
  unsigned dst[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = wave + 4 * i, row = 16 * j + (lane >> 2);
    gb[i] = B.B + (size_t)min(i0 + row, mp - 1) * mp + nt_chunk(row, lane & 3) * 8;
    const int k = XROWS * j + lane / XCH;
    const int sw = T == 128 ? 2 * (k & 7) : 2 * ((k >> 1) & 3);
    gx[i] = X + (size_t)k * np + min(j0 + ((lane % XCH) ^ sw) * 8, np - 8);
    dst[i] = j * 1024;
  }
  const unsigned base = lds_addr(sm);
  auto issue = [&](int kt, int buf) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      lds_dma16(gb[i] + kt * 32, base + buf * (STAGE * 2) + dst[i]);
      lds_dma16(gx[i] + (size_t)kt * 32 * np, base + buf * (STAGE * 2) + OP * 2 + dst[i]);
    }
  };
  f32x4 acc[WT][WT];  // [i][j]
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < WT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  int fb[WT], fx[WT];
  {
    const int r = 4 * lg + q4;  // the transposing read of k rows 4 lg .. and 16 + 4 lg ..: the swizzle is the same for both
    const int sw = T == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3);
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      const int rb = (wi * WT + i) * 16 + l15;
      fb[i] = rb * 32 + nt_chunk(rb, lg) * 8;
      const int lc = 2 * (wj * WT + i) + (p4 >> 1);
      fx[i] = OP + r * T + (lc ^ sw) * 8 + (p4 & 1) * 4;
    }
  }
  const bool along_i = MODE != MID && I.tall;
  const int nk = mp / 32;
#pragma unroll
  for (int st = 0; st < NB - 1; ++st)
    if (st < nk) issue(st, st);
  int buf = 0;
  for (int kt = 0; kt < nk; ++kt) {
    wait_stage<2 * PER, NB>(min(nk - 1 - kt, NB - 2));
    __syncthreads();
    if (kt + NB - 1 < nk) issue(kt + NB - 1, buf == 0 ? NB - 1 : buf - 1);
    const f16* s = sm + buf * STAGE;
    f16x8 vb[WT], vx[WT];
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      vb[i] = *reinterpret_cast<const f16x8*>(s + fb[i]);
      const f16x4 x0 = read_tr(s + fx[i]);
      const f16x4 x1 = read_tr(s + fx[i] + 16 * T);
      vx[i] = (f16x8){x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
    }
    if (along_i) {
#pragma unroll
      for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb[i], vx[j], acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < WT; ++i)
#pragma unroll
        for (int j = 0; j < WT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vx[j], vb[i], acc[i][j], 0, 0, 0);
    }
    buf = buf == NB - 1 ? 0 : buf + 1;
  }

  float* p = nullptr;
  if constexpr (MODE == STEP) p = mo.p_ptrs[I.index];
  const float step = MODE == STEP ? mo.lr * I.scale : 0.f;
  // four results x[r] of G's row `gr`, columns gc .. gc + 3
  auto put = [&](int gr, int gc, const float* x) {
    if (gr >= I.rows || gc >= I.cols) return;
    const int have = min(4, I.cols - gc);
    if constexpr (MODE == OUT) {
      if (otype == SWG_BF16) {
        bf16* d = (bf16*)I.dst + (int64_t)b * I.bs_dst + (int64_t)gr * I.ld_dst + gc;
        if (have == 4 && ((size_t)d & 7) == 0) *reinterpret_cast<uint2*>(d) = pack_bf16x4(x[0], x[1], x[2], x[3]);
        else
          for (int r = 0; r < have; ++r) d[r] = (bf16)x[r];
      } else {
        f16* d = (f16*)I.dst + (int64_t)b * I.bs_dst + (int64_t)gr * I.ld_dst + gc;
        if (have == 4 && ((size_t)d & 7) == 0) *reinterpret_cast<f16x4*>(d) = (f16x4){(f16)x[0], (f16)x[1], (f16)x[2], (f16)x[3]};
        else
          for (int r = 0; r < have; ++r) d[r] = (f16)x[r];
      }
    } else if constexpr (MODE == STEP) {
      const int64_t at = (int64_t)gr * I.cols + gc;
      float* pp = p + at;
      float* ee = mo.ema + I.flat_off + at;
      if (have == 4 && (((size_t)pp | (mo.n_ema ? (size_t)ee | (size_t)(mo.total * 4) : 0)) & 15) == 0) {
        float4 v = *reinterpret_cast<float4*>(pp);
        v.x = mo.keep * v.x - step * x[0]; v.y = mo.keep * v.y - step * x[1];
        v.z = mo.keep * v.z - step * x[2]; v.w = mo.keep * v.w - step * x[3];
        *reinterpret_cast<float4*>(pp) = v;
        for (int k = 0; k < mo.n_ema; ++k) {
          float4* e = reinterpret_cast<float4*>(ee + (int64_t)k * mo.total);
          float4 ev = *e;
          const float wk = mo.ema_w[k];
          ev.x += wk * (v.x - ev.x); ev.y += wk * (v.y - ev.y); ev.z += wk * (v.z - ev.z); ev.w += wk * (v.w - ev.w);
          *e = ev;
        }
      } else {
        for (int r = 0; r < have; ++r) {
          const float v = mo.keep * pp[r] - step * x[r];
          pp[r] = v;
          for (int k = 0; k < mo.n_ema; ++k) {
            float* e = ee + (int64_t)k * mo.total + r;
            *e += mo.ema_w[k] * (v - *e);
          }
        }
      }
    }
  };
  if (along_i) {
#pragma unroll
    for (int j = 0; j < WT; ++j) {
      const int jj = j0 + (wj * WT + j) * 16 + l15;
#pragma unroll
      for (int i = 0; i < WT; ++i) {
        const int ii = i0 + (wi * WT + i) * 16 + 4 * lg;
        if (ii >= mp || jj >= np) continue;
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const size_t at = (size_t)(ii + r) * np + jj;
          const float h = (float)X[at], l = (float)B.lo[at];
          x[r] = (QA * (h + l) + B.dB[ii + r] * h + acc[i][j][r] * (1.f / SB)) * (1.f / SX);
        }
        put(jj, ii, x);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < WT; ++i) {
      const int ii = i0 + (wi * WT + i) * 16 + l15;
      if (ii >= mp) continue;
      const float e = B.dB[ii];
#pragma unroll
      for (int j = 0; j < WT; ++j) {
        const int jj = j0 + (wj * WT + j) * 16 + 4 * lg;
        if (jj >= np) continue;
        const size_t at = (size_t)ii * np + jj;
        const f16x4 h4 = *reinterpret_cast<const f16x4*>(X + at), l4 = *reinterpret_cast<const f16x4*>(B.lo + at);
        float x[4];
        f16x4 nh, nl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float h = (float)h4[r];
          x[r] = QA * (h + (float)l4[r]) + e * h + acc[i][j][r] * (1.f / SB);
          nh[r] = (f16)x[r];
          nl[r] = (f16)(x[r] - (float)nh[r]);
          x[r] *= 1.f / SX;
        }
        if constexpr (MODE == MID) {
          *reinterpret_cast<f16x4*>(B.hi(cur ^ 1) + at) = nh;
          *reinterpret_cast<f16x4*>(B.lo + at) = nl;
        } else {
          put(ii, jj, x);
        }
      }
    }
  }
}

// sum of squares of all gradients in a fixed order: fp64 partial sums per workgroup, then one workgroup
__global__ __launch_bounds__(256) void k_sqnorm_parts(const float* const* __restrict__ g_ptrs,
                                                      const int32_t* __restrict__ numel,
                                                      const int32_t* __restrict__ chunk_tensor,
                                                      const int32_t* __restrict__ chunk_off, int n_chunks, int chunk,
                                                      double* __restrict__ part) {
  __shared__ double red[4];
  double s = 0.0;
  for (int c = blockIdx.x; c < n_chunks; c += gridDim.x) {
    const int t = chunk_tensor[c], off = chunk_off[c], n = min(chunk, numel[t] - off);
    const float* g = g_ptrs[t] + off;
    for (int i = threadIdx.x; i < n; i += 256) s += (double)g[i] * (double)g[i];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}
__global__ __launch_bounds__(256) void k_sqnorm_total(const double* __restrict__ part, int n, float* __restrict__ out) {
  __shared__ double red[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) s += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) *out = (float)((red[0] + red[1]) + (red[2] + red[3]));
}
constexpr int SQNORM_BLOCKS = 1024;

// ---- host ----------------------------------------------------------------------------------------------------------
// What a call over a list of shapes needs; the same arithmetic sizes the workspace, fills the table and sizes the grids
struct Plan {
  int count = 0, wt = 2;
  int64_t grid[PREFIXES] = {0, 0, 0, 0, 0};
  int64_t parts = 0;
  size_t bytes = 0;                            // of X, A, B and the diagonals of all matrices
  double flops = 0;
};

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

// tile side: 128 where that gives at least 1.5 workgroups a CU in the narrowest product, else 64
bool plan_item(Plan& P, int32_t rows, int32_t cols, int32_t batch, Item* I) {
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
  i.stride = (int64_t)align256((size_t)3 * i.mp * i.np * 2 + (size_t)2 * i.mp * i.mp * 2 + (size_t)2 * i.mp * 4);
  P.parts += (int64_t)i.batch * i.parts;
  P.bytes += (size_t)i.batch * (size_t)i.stride;
  P.flops += (double)i.batch * (3.0 * i.m * i.m * (double)i.n + (double)i.m * i.m * (double)i.m);
  P.count += 1;
  if (I) *I = i;
  return true;
}
void plan_grids(const Item& i, int wt, int64_t* g) {
  const int T = 32 * wt;
  const int64_t nt = cdiv64(i.mp, T), b = i.batch;
  g[P_NORM] += b * i.parts;
  g[P_INIT] += b * cdiv64(i.mp, INIT_TILE) * cdiv64(i.np, INIT_TILE);
  g[P_SYM] += b * (nt * (nt + 1) / 2);
  g[P_FULL] += b * nt * cdiv64(i.np, T);
}

// plan buffer (device): Item[count], int32 ends[PREFIXES][count], then the fp64 partial sums
size_t table_bytes(int count) { return align256((size_t)count * sizeof(Item)) + align256((size_t)count * PREFIXES * 4); }

template <class F>
bool make_plan(int32_t count, F shape, Plan& P) {  // shape(i, rows, cols, batch)
  if (count < 0) return false;
  int64_t big = 0;
  for (int pass = 0; pass < 2; ++pass) {
    P.parts = 0; P.bytes = 0; P.flops = 0; P.count = 0;
    for (int k = 0; k < PREFIXES; ++k) P.grid[k] = 0;
    for (int32_t i = 0; i < count; ++i) {
      int32_t r, c, b;
      shape(i, r, c, b);
      Item it;
      if (!plan_item(P, r, c, b, &it)) return false;
      plan_grids(it, pass == 0 ? 4 : P.wt, P.grid);
    }
    if (pass == 0) {
      big = P.grid[P_SYM];
      P.wt = big >= 384 ? 4 : 2;
    }
  }
  for (int k = 0; k < PREFIXES; ++k)
    if (P.grid[k] > 0x7fffffff) return false;
  return true;
}

template <class F>
int write_table(int32_t count, const Plan& P, F fill, void* table, hipStream_t s) {  // fill(i, item): the caller's fields
  Item* items = (Item*)table;
  int32_t* ends = (int32_t*)((char*)table + align256((size_t)count * sizeof(Item)));
  Plan run;
  int64_t g[PREFIXES] = {0, 0, 0, 0, 0};
  for (int first = 0; first < count; first += TABLE_BATCH) {
    EntryBatch eb;
    const int n = count - first < TABLE_BATCH ? count - first : TABLE_BATCH;
    for (int k = 0; k < n; ++k) {
      fill(first + k, run, eb.e[k].item);
      plan_grids(eb.e[k].item, P.wt, g);
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
  char* ws;
  int count;
  const int32_t* end(int k) const { return ends + (size_t)k * count; }
};
size_t ws_bytes_of(const Plan& P) { return align256((size_t)P.parts * 8) + P.bytes; }
Ptrs ptrs_of(int count, const Plan& P, const void* table, void* ws) {
  Ptrs r;
  r.items = (const Item*)table;
  r.ends = (const int32_t*)((const char*)table + align256((size_t)count * sizeof(Item)));
  r.part = (double*)ws;
  r.ws = (char*)ws + align256((size_t)P.parts * 8);
  r.count = count;
  return r;
}

template <int MODE, int WT, int NB>
int run_steps(const Plan& P, const Ptrs& p, int steps, int otype, const Momentum& mo, hipStream_t s) {
  const dim3 gs((unsigned)P.grid[P_SYM]), gf((unsigned)P.grid[P_FULL]);
  int cur = 0;
  for (int k = 0; k < steps; ++k) {
    hipLaunchKernelGGL((k_orth_sym<true, WT, NB>), gs, dim3(256), 0, s, p.items, p.end(P_SYM), p.count, cur, p.ws);
    hipLaunchKernelGGL((k_orth_sym<false, WT, NB>), gs, dim3(256), 0, s, p.items, p.end(P_SYM), p.count, cur, p.ws);
    if (k + 1 < steps)
      hipLaunchKernelGGL((k_orth_apply<MID, WT, NB>), gf, dim3(256), 0, s, p.items, p.end(P_FULL), p.count, cur, otype,
                         p.ws, mo);
    else
      hipLaunchKernelGGL((k_orth_apply<MODE, WT, NB>), gf, dim3(256), 0, s, p.items, p.end(P_FULL), p.count, cur, otype,
                         p.ws, mo);
    SWG_LAUNCH_CHECK();
    cur ^= 1;
  }
  return 0;
}
template <int MODE>
int run_steps(const Plan& P, const Ptrs& p, int steps, int otype, const Momentum& mo, hipStream_t s) {
  return P.wt == 4 ? run_steps<MODE, 4, 3>(P, p, steps, otype, mo, s) : run_steps<MODE, 2, 4>(P, p, steps, otype, mo, s);
}

template <class T, bool MOM>
int run_init(const Plan& P, const Ptrs& p, float eps, const Momentum& mo, hipStream_t s) {
  hipLaunchKernelGGL((k_orth_norm<T, MOM>), dim3((unsigned)P.grid[P_NORM]), dim3(256), 0, s, p.items, p.end(P_NORM), p.count,
                     p.part, mo);
  SWG_LAUNCH_CHECK();
  hipLaunchKernelGGL((k_orth_init<T, MOM>), dim3((unsigned)P.grid[P_INIT]), dim3(256), 0, s, p.items, p.end(P_INIT), p.count,
                     p.part, (double)eps, p.ws, mo);
  SWG_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" {

size_t swg_orthogonalise_workspace_bytes(int32_t count, const swg_orth_item* items) {
  if (count <= 0 || !items) return 0;
  Plan P;
  if (!make_plan(count, [&](int i, int32_t& r, int32_t& c, int32_t& b) { r = items[i].rows; c = items[i].cols; b = items[i].batch; }, P))
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
  if (!make_plan(count, [&](int i, int32_t& r, int32_t& c, int32_t& b) { r = items[i].rows; c = items[i].cols; b = items[i].batch; }, P))
    return SWG_E_SHAPE;
  for (int i = 0; i < count; ++i) {
    const swg_orth_item& e = items[i];
    if (e.rows == 0 || e.cols == 0 || e.batch == 0) continue;
    if (!e.g || !e.out) return SWG_E_NULL;
    if (e.ld_g < e.cols || e.ld_out < e.cols) return SWG_E_SHAPE;
  }
  if (P.grid[P_FULL] == 0) return 0;
  if (!ws) return SWG_E_NULL;
  if (ws_bytes < table_bytes(count) + ws_bytes_of(P) + 256) return SWG_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  void* table = (void*)(((size_t)ws + 255) & ~(size_t)255);
  SwgProfScope ps(KID_ORTH, P.flops * steps, 0.0, s);
  int r = write_table(count, P, [&](int i, Plan& run, Item& I) {
    const swg_orth_item& e = items[i];
    plan_item(run, e.rows, e.cols, e.batch, &I);
    I.src = e.g; I.dst = e.out; I.ld_src = e.ld_g; I.bs_src = e.bs_g; I.ld_dst = e.ld_out; I.bs_dst = e.bs_out;
  }, table, s);
  if (r) return r;
  const Ptrs p = ptrs_of(count, P, table, (char*)table + table_bytes(count));
  const Momentum none = {};
  if (itype == SWG_F32) r = run_init<float, false>(P, p, eps, none, s);
  else if (itype == SWG_BF16) r = run_init<bf16, false>(P, p, eps, none, s);
  else r = run_init<f16, false>(P, p, eps, none, s);
  if (r) return r;
  return run_steps<OUT>(P, p, steps, otype, none, s);
}

static bool muon_plan(int32_t count, const swg_muon_item* items, Plan& P) {
  return make_plan(count, [&](int i, int32_t& r, int32_t& c, int32_t& b) { r = items[i].rows; c = items[i].cols; b = 1; }, P);
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
  if (table_size < table_bytes(count)) return SWG_E_WORKSPACE;
  return write_table(count, P, [&](int i, Plan& run, Item& I) {
    plan_item(run, items[i].rows, items[i].cols, 1, &I);
    I.flat_off = items[i].flat_off; I.index = items[i].index; I.scale = items[i].scale;
  }, table, (hipStream_t)stream);
}

int swg_muon_ema_step(int32_t count, const swg_muon_item* items, const void* table, const void* p_ptrs, const void* g_ptrs,
                      float* m, float* ema, int64_t total, int32_t n_ema, const float* ema_decay, const float* sqnorm,
                      float max_norm, float lr, float momentum, int32_t nesterov, float weight_decay, int32_t steps,
                      float eps, void* ws, size_t ws_bytes, void* stream) {
  if (count <= 0 || total <= 0 || n_ema < 0 || n_ema > 8 || steps < 1 || steps > 64 || !(eps >= 0.f)) return SWG_E_SHAPE;
  if (!items || !table || !p_ptrs || !g_ptrs || !m || !ws || (n_ema > 0 && (!ema || !ema_decay))) return SWG_E_NULL;
  Plan P;
  if (!muon_plan(count, items, P)) return SWG_E_SHAPE;
  if (ws_bytes < ws_bytes_of(P)) return SWG_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  Momentum mo = {};
  mo.g_ptrs = (const float* const*)g_ptrs; mo.p_ptrs = (float* const*)p_ptrs;
  mo.m = m; mo.ema = ema; mo.total = total; mo.sqnorm = sqnorm; mo.max_norm = max_norm; mo.mu = momentum; mo.lr = lr;
  mo.keep = 1.f - lr * weight_decay; mo.nesterov = nesterov; mo.n_ema = n_ema;
  for (int k = 0; k < n_ema; ++k) mo.ema_w[k] = 1.0f - ema_decay[k];
  SwgProfScope ps(KID_ORTH, P.flops * steps, 0.0, s);
  const Ptrs p = ptrs_of(count, P, table, ws);
  if (int r = run_init<float, true>(P, p, eps, mo, s)) return r;
  return run_steps<STEP>(P, p, steps, 0, mo, s);
}

size_t swg_grad_sqnorm_ordered_workspace_bytes(void) { return SQNORM_BLOCKS * sizeof(double); }

int swg_grad_sqnorm_ordered(const void* g_ptrs, const int32_t* numel, const int32_t* chunk_tensor, const int32_t* chunk_off,
                            int32_t n_chunks, float* sqnorm, void* ws, size_t ws_bytes, void* stream) {
  if (!g_ptrs || !numel || !chunk_tensor || !chunk_off || !sqnorm || !ws) return SWG_E_NULL;
  if (n_chunks <= 0) return SWG_E_SHAPE;
  if (ws_bytes < SQNORM_BLOCKS * sizeof(double)) return SWG_E_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const int grid = n_chunks < SQNORM_BLOCKS ? n_chunks : SQNORM_BLOCKS;
  SwgProfScope ps(KID_OPTIM, 0.0, 0.0, s);
  hipLaunchKernelGGL(k_sqnorm_parts, dim3(grid), dim3(256), 0, s, (const float* const*)g_ptrs, numel, chunk_tensor, chunk_off,
                     n_chunks, swg_optim_chunk(), (double*)ws);
  hipLaunchKernelGGL(k_sqnorm_total, dim3(1), dim3(256), 0, s, (const double*)ws, grid, sqnorm);
  SWG_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
