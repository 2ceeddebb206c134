// Newton-Schulz orthogonalisation of many matrices at once, and the Muon optimizer step built on it.
//
// For G [rows, cols], s = min(rows, cols), l = max: X = G (or its transpose: s x l) / max(|G|_F, eps), then `steps` times
//     A = X X^T      R = b A + c A A      X <- a X + R X
// The three products are matrix-core work; everything else rides in their epilogues.
//
// Arithmetic: the iteration multiplies rounding errors by up to a^steps (485 at the usual coefficients), so 8 or 11 bit
// operands lose the small directions of G.  Every operand is therefore kept as TWO fp16 numbers, x = hi + lo (hi = x rounded
// to fp16, lo = the rest rounded to fp16: together 22 bits, 2^-23 of the value at worst), and a product is three fp16 matrix
// instructions, hi hi + hi lo + lo hi, summed in fp32; the missing lo lo is below 2^-22 of the product.  Measured on the CPU
// the result is as far from the 64-bit one as an fp32 iteration is.  fp16 holds the range because X, A, R and their products
// are bounded (|X| <= 1.3 or so, |R| <= 5 at the usual coefficients; other coefficients are checked on the host): they
// are stored times 2^11, which leaves values down to 2^-25 of the largest their full 22 bits.
//
// Storage: a matrix [R, K] (both padded with zeros to multiples of 128) holds, per row and 32 columns, 64 bytes of hi and 64
// bytes of lo: 128-byte lines that are exactly one K-step of a tile row.  A and R are symmetric: only their tiles on and
// above the diagonal are computed, the others are written as mirror images.
#include "common.h"

typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) _Float16 f16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef s16x4 __attribute__((address_space(3))) * lds_s16x4;

#define NS_PAD 128                 // both axes of a stored matrix
#define NS_SCALE 2048.f            // stored value = 2^11 x
#define NS_CHUNK 16384             // elements a workgroup of the norm pass reads
#define NS_MAX_SHORT 16384
#define NS_MAX_LONG (1 << 22)

// One matrix.  Offsets into the user's buffers are in elements, into the workspace in bytes.
struct NsMat {
  long at;                         // first element, row-major [rows, cols]
  int rows, cols;
  int s, l, sp, lp;                // short / long side, padded
  int tall, parts;                 // rows > cols; number of norm partials
  float scale, pad_;
  long x, sq, norm;                // X (two buffers of 4 sp lp bytes), squares (four of 4 sp sp), partials (doubles)
};

// What every kernel here gets: the matrices, the tiles, the workspace.  `list` (plan): (matrix, ti, tj, 0) per workgroup;
// without it every matrix looks like `one` and workgroups are numbered matrix by matrix.
struct NsGroup {
  const NsMat* mats;
  NsMat one;
  long ws_stride, at_stride;       // bytes / elements from one matrix of the batch to the next
  unsigned char* ws;
};
struct NsTile { int mat, ti, tj; };

__device__ __forceinline__ NsMat ns_mat(const NsGroup& g, int mat) {
  if (g.mats) return g.mats[mat];
  NsMat m = g.one;
  m.at += mat * g.at_stride;
  m.x += mat * g.ws_stride;
  m.sq += mat * g.ws_stride;
  m.norm += mat * g.ws_stride;
  return m;
}

__device__ __forceinline__ void ns_split(float v, _Float16& hi, _Float16& lo) {      // v already scaled
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

template <int N> __device__ __forceinline__ void ns_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// 64 lanes x 16 bytes, per-lane global address -> LDS [addr + 16 lane]; addr is wave-uniform.  In asm so that the compiler's
// waits for the fragment reads stay counted ones; ordered by the explicit vmcnt waits and barriers.
__device__ __forceinline__ void ns_dma(const void* src, unsigned lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds_addr)), "v"(src)
               : "memory");
}
__device__ __forceinline__ unsigned ns_lds(const void* p) { return (unsigned)(uintptr_t)(lptr_t)p; }

// ------------------------------------------------------------------------------------------------ norm, momentum, split
struct NsSource {
  const void* src;                 // orthogonalize: the matrices, fp32 or bf16
  float *g, *m;                    // Muon: gradient and momentum
  float mu, rest, grad_scale;      // rest = 1 - mu, formed in 64 bits by the caller
  int nesterov, zero_grad, bf16;
  float eps;
};

// Partial sums of squares in 64 bits (no gradient is too small or too large), one per NS_CHUNK elements.  Muon: the momentum
// update M <- mu M + (1 - mu) g on the way, and the squares are those of U = (1 - mu) g + mu M (Nesterov) or M.
template <int KIND>                // 0 fp32, 1 bf16, 2 Muon
__global__ __launch_bounds__(256) void ns_norm_kernel(NsGroup grp, NsSource q, const int* __restrict__ chunks, int per) {
  int mat, chunk;
  if (chunks) { mat = chunks[2 * blockIdx.x]; chunk = chunks[2 * blockIdx.x + 1]; }
  else { mat = blockIdx.x / per; chunk = blockIdx.x - mat * per; }
  const NsMat M = ns_mat(grp, mat);
  const long n = (long)M.rows * M.cols, lo = (long)chunk * NS_CHUNK, hi = min(n, lo + NS_CHUNK);
  double sum = 0.0;
  for (long e = lo + threadIdx.x; e < hi; e += 256) {
    float v;
    if constexpr (KIND == 2) {
      const float g = q.g[M.at + e] * q.grad_scale, m = q.mu * q.m[M.at + e] + q.rest * g;
      q.m[M.at + e] = m;
      v = q.nesterov ? q.rest * g + q.mu * m : m;
    } else {
      v = KIND == 1 ? to_f32(((const bf16_t*)q.src)[M.at + e]) : ((const float*)q.src)[M.at + e];
    }
    sum += (double)v * (double)v;
  }
  __shared__ double lds[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) ((double*)(grp.ws + M.norm))[chunk] = lds[0] + lds[1] + lds[2] + lds[3];
}

// X0 = U / max(|U|, eps) in split form, padding included; a 64 x 64 piece of X a workgroup, through LDS so that the source is
// read along its rows in both orientations.
template <int KIND>
__global__ __launch_bounds__(256) void ns_split_kernel(NsGroup grp, NsSource q, const int* __restrict__ list, int per) {
  NsTile t;
  const int tile = blockIdx.x >> 2, piece = blockIdx.x & 3;          // four pieces of a 128 x 128 tile
  if (list) { t.mat = list[4 * tile]; t.ti = list[4 * tile + 1]; t.tj = list[4 * tile + 2]; }
  else {
    t.mat = tile / per;
    const int r = tile - t.mat * per, nj = grp.one.lp / NS_PAD;
    t.ti = r / nj;
    t.tj = r - t.ti * nj;
  }
  const NsMat M = ns_mat(grp, t.mat);
  __shared__ float tilebuf[64][65];
  __shared__ double part[4];
  double sum = 0.0;
  const double* parts = (const double*)(grp.ws + M.norm);
  for (int i = threadIdx.x; i < M.parts; i += 256) sum += parts[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  const double norm = sqrt(part[0] + part[1] + part[2] + part[3]);
  const float inv = (float)((double)NS_SCALE / (norm > (double)q.eps ? norm : (norm <= (double)q.eps ? (double)q.eps : norm)));
  const int i0 = t.ti * 128 + (piece >> 1) * 64, j0 = t.tj * 128 + (piece & 1) * 64;   // X rows (short side), columns
  const int c = threadIdx.x & 63;
#pragma unroll 4
  for (int k = threadIdx.x >> 6; k < 64; k += 4) {
    const int r = M.tall ? j0 + k : i0 + k, col = M.tall ? i0 + c : j0 + c;            // in the user's orientation
    float v = 0.f;
    if (r < M.rows && col < M.cols) {
      const long e = M.at + (long)r * M.cols + col;
      if constexpr (KIND == 2) {
        const float m = q.m[e];
        v = q.nesterov ? q.rest * (q.g[e] * q.grad_scale) + q.mu * m : m;
        if (q.zero_grad) q.g[e] = 0.f;
      } else {
        v = KIND == 1 ? to_f32(((const bf16_t*)q.src)[e]) : ((const float*)q.src)[e];
      }
      v *= inv;
    }
    if (M.tall) tilebuf[c][k] = v;
    else tilebuf[k][c] = v;
  }
  __syncthreads();
  unsigned char* X = grp.ws + M.x;
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int item = threadIdx.x + 256 * u, row = item >> 3, g8 = item & 7;
    f16x8 hi, lo;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      _Float16 h, l;
      ns_split(tilebuf[row][g8 * 8 + e], h, l);
      hi[e] = h;
      lo[e] = l;
    }
    const int col = j0 + g8 * 8;
    unsigned char* o = X + (size_t)(i0 + row) * M.lp * 4 + (col >> 5) * 128 + (col & 31) * 2;
    *(f16x8*)o = hi;
    *(f16x8*)(o + 64) = lo;
  }
}

// ------------------------------------------------------------------------------------------------ products
enum { NS_GRAM = 0, NS_SQUARE = 1, NS_APPLY = 2 };
enum { NS_OUT_PLANES = 0, NS_OUT_F32 = 1, NS_OUT_BF16 = 2, NS_OUT_MUON = 3 };

struct NsProduct {
  int a, b, e1, e2, out;           // square buffers (SQUARE: A, B^T = B; addends; result) / X buffer read and written (APPLY: b, out)
  float ca, c1, c2;                // result = ca A B + c1 E1 + c2 E2
  void* dst;                       // last APPLY: the user's buffer
  float *p, *ema;                  // Muon
  bf16_t* shadow;
  float decay, lr, ema_beta, ema_rest;   // W <- decay W - lr scale O
  int do_ema;
  const int* state;
};

// Tile BM x BN by WM x WN waves.  K-steps of 32: A tile [BM][hi 64 B | lo 64 B], B tile the same (products with a
// symmetric or transposed right side) or, for R X, [32 rows of X][BN columns], read by the transposing LDS read.  D LDS stages
// filled by asynchronous loads: step k waits (counted) for its own, passes one barrier, sends stage k + D - 1 on its way into the
// buffer that step k - 1 has finished with, and multiplies.
template <int KIND, int BM, int BN, int WM, int WN, int D, int OUT>
__global__ __launch_bounds__(64 * WM * WN) void ns_product_kernel(NsGroup grp, NsProduct q, const int* __restrict__ list,
                                                                   int per) {
  constexpr int NW = WM * WN, MI = BM / WM / 16, NJ = BN / WN / 16;
  constexpr int A_BYTES = BM * 128, STAGE = (BM + BN) * 128;
  constexpr int AP = BM / 8 / NW, BP = BN / 8 / NW, PIECES = AP + BP;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "whole pieces a wave");
  __shared__ __attribute__((aligned(1024))) unsigned char smem[D * STAGE];
  NsTile t;
  if (list) { t.mat = list[4 * blockIdx.x]; t.ti = list[4 * blockIdx.x + 1]; t.tj = list[4 * blockIdx.x + 2]; }
  else {
    t.mat = blockIdx.x / per;
    int r = blockIdx.x - t.mat * per;
    if constexpr (KIND == NS_APPLY) {
      const int nj = grp.one.lp / BN;
      t.ti = r / nj;
      t.tj = r - t.ti * nj;
    } else {
      const int n = grp.one.sp / BM;
      t.ti = 0;
      while (r >= n - t.ti) { r -= n - t.ti; t.ti++; }
      t.tj = t.ti + r;
    }
  }
  const NsMat M = ns_mat(grp, t.mat);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave - wm * WN;
  const size_t sq = (size_t)M.sp * M.sp * 4, xs = (size_t)M.sp * M.lp * 4;
  const unsigned char *Ap, *Bp;
  size_t lda, ldb;
  int K;
  if constexpr (KIND == NS_GRAM) { Ap = Bp = grp.ws + M.x + q.b * xs; lda = ldb = (size_t)M.lp * 4; K = M.lp; }
  else if constexpr (KIND == NS_SQUARE) {
    Ap = grp.ws + M.sq + q.a * sq;
    Bp = grp.ws + M.sq + q.b * sq;
    lda = ldb = (size_t)M.sp * 4;
    K = M.sp;
  } else {
    Ap = grp.ws + M.sq + q.a * sq;
    Bp = grp.ws + M.x + q.b * xs;
    lda = (size_t)M.sp * 4;
    ldb = (size_t)M.lp * 4;
    K = M.sp;
  }
  const int i0 = t.ti * BM, j0 = t.tj * BN;
  // source addresses of this lane's pieces for K-step 0; the LDS image is lane-linear, so the bank swizzle (chunk ^= row & 7;
  // for the X rows a 32-byte swizzle that puts the 8 rows a half wave reads into different banks) is done on the source side
  const unsigned char *asrc[AP], *bsrc[BP];
#pragma unroll
  for (int j = 0; j < AP; j++) {
    const int row = (wave * AP + j) * 8 + (lane >> 3);
    asrc[j] = Ap + (size_t)(i0 + row) * lda + (((lane & 7) ^ (row & 7)) << 4);
  }
  constexpr int RB = BN * 4;                                  // bytes of a row of the X tile
#pragma unroll
  for (int j = 0; j < BP; j++) {
    if constexpr (KIND == NS_APPLY) {
      const int at = (wave * BP + j) * 1024 + lane * 16, row = at / RB, chunk = (at - row * RB) >> 4;
      const int z = (row & 3) | ((row >> 3) & 1) << 2;
      bsrc[j] = Bp + (size_t)row * ldb + (size_t)j0 * 4 + ((chunk ^ (z << 1)) << 4);
    } else {
      const int row = (wave * BP + j) * 8 + (lane >> 3);
      bsrc[j] = Bp + (size_t)(j0 + row) * ldb + (((lane & 7) ^ (row & 7)) << 4);
    }
  }
  const size_t bstep = KIND == NS_APPLY ? 32 * ldb : 128;
  const int nsteps = K >> 5;
  auto issue = [&](int step) {
    unsigned char* base = &smem[(step % D) * STAGE];
#pragma unroll
    for (int j = 0; j < AP; j++) ns_dma(asrc[j] + (size_t)step * 128, ns_lds(base + (wave * AP + j) * 1024));
#pragma unroll
    for (int j = 0; j < BP; j++) ns_dma(bsrc[j] + (size_t)step * bstep, ns_lds(base + A_BYTES + (wave * BP + j) * 1024));
  };
  f32x4 acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int fr = lane & 15, fq = lane >> 4, tq = fr >> 2, tp = fr & 3;
#pragma unroll
  for (int d = 0; d < D - 1; d++)
    if (d < nsteps) issue(d);
  for (int k = 0; k < nsteps; k++) {
    if (k + D - 1 <= nsteps) ns_wait_vm<(D - 2) * PIECES>();
    else ns_wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    const unsigned char* As = &smem[(k % D) * STAGE];
    const unsigned char* Bs = As + A_BYTES;
    f16x8 ah[MI], al[MI], bh[NJ], bl[NJ];
#pragma unroll
    for (int i = 0; i < MI; i++) {
      const int ra = wm * (BM / WM) + i * 16 + fr;
      ah[i] = *(const f16x8*)(As + ra * 128 + ((fq ^ (ra & 7)) << 4));
      al[i] = *(const f16x8*)(As + ra * 128 + (((fq + 4) ^ (ra & 7)) << 4));
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      if constexpr (KIND == NS_APPLY) {
        const int r0 = 8 * fq + tq, z = (r0 & 3) | ((r0 >> 3) & 1) << 2;    // (the same for row r0 + 4)
        const int cb = wn * (BN / WN / 16) + j, c = (cb >> 1) * 8 + (cb & 1) * 2 + (tp >> 1), o = 8 * (tp & 1);
        const unsigned char* h0 = Bs + r0 * RB + ((c ^ (z << 1)) << 4) + o;
        const unsigned char* l0 = Bs + r0 * RB + (((c + 4) ^ (z << 1)) << 4) + o;
        const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)h0);
        const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(h0 + 4 * RB));
        const s16x4 b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)l0);
        const s16x4 b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(l0 + 4 * RB));
        bh[j] = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
        bl[j] = __builtin_bit_cast(f16x8, (s16x8)__builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
      } else {
        const int rb = wn * (BN / WN) + j * 16 + fr;
        bh[j] = *(const f16x8*)(Bs + rb * 128 + ((fq ^ (rb & 7)) << 4));
        bl[j] = *(const f16x8*)(Bs + rb * 128 + (((fq + 4) ^ (rb & 7)) << 4));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (k + D - 1 < nsteps) issue(k + D - 1);
    __builtin_amdgcn_sched_barrier(0);
    // operands swapped: a lane then holds four consecutive columns of one row
#pragma unroll
    for (int i = 0; i < MI; i++)
#pragma unroll
      for (int j = 0; j < NJ; j++) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[j], ah[i], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], al[i], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], ah[i], acc[i][j], 0, 0, 0);
      }
  }

  // ---- epilogue, in units of the stored scale
  const float ca = q.ca * (1.f / NS_SCALE);
  const unsigned char *e1 = nullptr, *e2 = nullptr;
  size_t lde;
  unsigned char* out;
  if constexpr (KIND == NS_APPLY) {
    e1 = grp.ws + M.x + q.b * xs;
    lde = (size_t)M.lp * 4;
    out = grp.ws + M.x + q.out * xs;
  } else {
    if (KIND == NS_SQUARE) {
      e1 = grp.ws + M.sq + q.e1 * sq;
      if (q.e2 >= 0) e2 = grp.ws + M.sq + q.e2 * sq;
    }
    lde = (size_t)M.sp * 4;
    out = grp.ws + M.sq + q.out * sq;
  }
  const bool mirror = KIND != NS_APPLY && t.ti != t.tj;
  int do_ema = 0;
  if constexpr (OUT == NS_OUT_MUON) do_ema = q.state ? q.state[1] : q.do_ema;
  auto addend = [&](const unsigned char* e, int m, int n) {
    const unsigned char* a = e + (size_t)m * lde + (n >> 5) * 128 + (n & 31) * 2;
    const f16x4 h = *(const f16x4*)a, l = *(const f16x4*)(a + 64);
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; r++) v[r] = (float)h[r] + (float)l[r];
    return v;
  };
#pragma unroll
  for (int i = 0; i < MI; i++)
#pragma unroll
    for (int j = 0; j < NJ; j++) {
      const int m = i0 + wm * (BM / WM) + i * 16 + fr, n = j0 + wn * (BN / WN) + j * 16 + 4 * fq;
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; r++) v[r] = ca * acc[i][j][r];
      if (KIND != NS_GRAM) {
        const f32x4 w = addend(e1, m, n);
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] += q.c1 * w[r];
      }
      if (KIND == NS_SQUARE && e2) {
        const f32x4 w = addend(e2, m, n);
#pragma unroll
        for (int r = 0; r < 4; r++) v[r] += q.c2 * w[r];
      }
      if constexpr (OUT == NS_OUT_PLANES) {
        f16x4 h, l;
#pragma unroll
        for (int r = 0; r < 4; r++) {
          _Float16 hh, ll;
          ns_split(v[r], hh, ll);
          h[r] = hh;
          l[r] = ll;
        }
        unsigned char* o = out + (size_t)m * lde + (n >> 5) * 128 + (n & 31) * 2;
        *(f16x4*)o = h;
        *(f16x4*)(o + 64) = l;
        if (mirror)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            unsigned char* om = out + (size_t)(n + r) * lde + (m >> 5) * 128 + (m & 31) * 2;
            *(_Float16*)om = h[r];
            *(_Float16*)(om + 64) = l[r];
          }
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int row = M.tall ? n + r : m, col = M.tall ? m : n + r;
          if (row >= M.rows || col >= M.cols) continue;
          const long e = M.at + (long)row * M.cols + col;
          const float o = v[r] * (1.f / NS_SCALE);
          if constexpr (OUT == NS_OUT_F32) ((float*)q.dst)[e] = o;
          else if constexpr (OUT == NS_OUT_BF16) ((bf16_t*)q.dst)[e] = (bf16_t)o;
          else {
            const float w = q.decay * q.p[e] - q.lr * M.scale * o;
            q.p[e] = w;
            if (q.shadow) q.shadow[e] = (bf16_t)w;
            if (do_ema == 1) q.ema[e] = q.ema_beta * q.ema[e] + q.ema_rest * w;
            else if (do_ema == 2) q.ema[e] = w;
          }
        }
      }
    }
}

// ------------------------------------------------------------------------------------------------ host
struct NsPlan {                    // start of a plan; lists and matrices follow
  long magic, bytes, ws_bytes, need;      // need: elements the flat buffers must have
  int mats, chunks, tri, full;
  long at_mats, at_chunks, at_gram, at_square, at_full;
};
static const long NS_MAGIC = 0x6d7501;

static inline int ns_up(int v) { return (v + NS_PAD - 1) / NS_PAD * NS_PAD; }
static bool ns_describe(NsMat& m, long at, int rows, int cols, float scale, long& ws) {
  if (rows < 1 || cols < 1 || at < 0) return false;
  m.at = at;
  m.rows = rows;
  m.cols = cols;
  m.tall = rows > cols;
  m.s = m.tall ? cols : rows;
  m.l = m.tall ? rows : cols;
  if (m.s > NS_MAX_SHORT || m.l > NS_MAX_LONG) return false;
  m.sp = ns_up(m.s);
  m.lp = ns_up(m.l);
  const long parts = ((long)rows * cols + NS_CHUNK - 1) / NS_CHUNK;
  m.parts = (int)parts;
  m.scale = scale;
  m.pad_ = 0.f;
  m.x = ws;
  ws += 2L * m.sp * m.lp * 4;
  m.sq = ws;
  ws += 4L * m.sp * m.sp * 4;
  m.norm = ws;
  ws += (parts * 8 + 255) / 256 * 256;
  return true;
}

struct NsRun {                     // one call: the group, its lists, its launch sizes
  NsGroup grp;
  const int *chunks, *gram, *square, *full;
  int n_chunks, n_tri, n_full;     // workgroups over all matrices
  int per_chunks, per_tri, per_full;
};

template <int KIND, int OUT>
static void ns_launch(const NsRun& r, const NsProduct& q, hipStream_t st) {
  const int* list = KIND == NS_APPLY ? r.full : KIND == NS_GRAM ? r.gram : r.square;
  hipLaunchKernelGGL((ns_product_kernel<KIND, 128, 128, 2, 2, 2, OUT>), dim3(KIND == NS_APPLY ? r.n_full : r.n_tri), dim3(256), 0,
                     st, r.grp, q, list, KIND == NS_APPLY ? r.per_full : r.per_tri);
}

// out: NS_OUT_F32 / BF16 / MUON for the last product; `last` holds its destination
static int ns_iterate(const NsRun& r, int steps, float a, float b, float c, int out, const NsProduct& last, hipStream_t st) {
  enum { G = 0, R = 1 };
  int x = 0;
  for (int k = 0; k < steps; k++) {
    NsProduct q = {};
    q.b = x;
    q.out = G;
    q.ca = 1.f;
    q.e2 = -1;
    ns_launch<NS_GRAM, NS_OUT_PLANES>(r, q, st);
    q.a = q.b = q.e1 = G;
    q.out = R;
    q.ca = c;
    q.c1 = b;
    ns_launch<NS_SQUARE, NS_OUT_PLANES>(r, q, st);
    q = k == steps - 1 ? last : q;
    q.a = R;
    q.b = x;
    q.out = x ^ 1;
    q.ca = 1.f;
    q.c1 = a;
    q.e2 = -1;
    if (k < steps - 1) ns_launch<NS_APPLY, NS_OUT_PLANES>(r, q, st);
    else if (out == NS_OUT_F32) ns_launch<NS_APPLY, NS_OUT_F32>(r, q, st);
    else if (out == NS_OUT_BF16) ns_launch<NS_APPLY, NS_OUT_BF16>(r, q, st);
    else ns_launch<NS_APPLY, NS_OUT_MUON>(r, q, st);
    x ^= 1;
    MADIFF_CHECK_LAUNCH();
  }
  return 0;
}

// The polynomial's orbit from every start in [0, 1]: the largest |x|, |A| and |R| on it have to stay in the stored range.
static bool ns_bounded(int steps, float a, float b, float c) {
  const double top = 65504.0 / NS_SCALE / 2;
  for (int i = 0; i <= 4096; i++) {
    double x = (double)i / 4096;
    for (int k = 0; k < steps; k++) {
      const double g = x * x, q = b * g + c * g * g;
      x = x * (a + q);
      if (!(x < top && x > -top && g < top && q < top && q > -top)) return false;
    }
  }
  return true;
}

extern "C" int madiff_ortho_check(int steps, float a, float b, float c, float eps) {
  return steps >= 1 && steps <= 64 && eps > 0.f && eps < 1e30f && ns_bounded(steps, a, b, c) ? 0 : -1;
}

extern "C" int madiff_ortho_ws(int batch, int rows, int cols, long* ws_bytes) {
  NsMat m;
  long ws = 0;
  if (batch < 0 || !ws_bytes || !ns_describe(m, 0, rows, cols, 1.f, ws)) return -1;
  const long tiles = (long)(m.sp / NS_PAD) * (m.lp / NS_PAD);
  if (batch > 0 && (tiles * 4 > 0x7fffffffL / batch || m.parts > 0x7fffffffL / batch)) return -1;
  *ws_bytes = ws * batch;
  return 0;
}

extern "C" int madiff_orthogonalize(int dtype, const void* src, void* dst, int batch, int rows, int cols, int steps, float a,
                                    float b, float c, float eps, void* ws, long ws_bytes, hipStream_t stream) {
  long need = 0;
  if ((dtype != MADIFF_F32 && dtype != MADIFF_BF16) || madiff_ortho_ws(batch, rows, cols, &need) ||
      madiff_ortho_check(steps, a, b, c, eps))
    return -1;
  if (batch == 0) return 0;
  if (!src || !dst || !ws || ws_bytes < need || ((size_t)ws & 255)) return -1;
  NsRun r = {};
  long stride = 0;
  ns_describe(r.grp.one, 0, rows, cols, 1.f, stride);
  const NsMat& m = r.grp.one;
  r.grp.ws_stride = stride;
  r.grp.at_stride = (long)rows * cols;
  r.grp.ws = (unsigned char*)ws;
  const int ni = m.sp / NS_PAD;
  r.per_chunks = m.parts;
  r.per_tri = ni * (ni + 1) / 2;
  r.per_full = ni * (m.lp / NS_PAD);
  r.n_chunks = batch * r.per_chunks;
  r.n_tri = batch * r.per_tri;
  r.n_full = batch * r.per_full;
  NsSource q = {};
  q.src = src;
  q.eps = eps;
  if (dtype == MADIFF_BF16) {
    hipLaunchKernelGGL((ns_norm_kernel<1>), dim3(r.n_chunks), dim3(256), 0, stream, r.grp, q, (const int*)nullptr, r.per_chunks);
    hipLaunchKernelGGL((ns_split_kernel<1>), dim3(4 * r.n_full), dim3(256), 0, stream, r.grp, q, (const int*)nullptr, r.per_full);
  } else {
    hipLaunchKernelGGL((ns_norm_kernel<0>), dim3(r.n_chunks), dim3(256), 0, stream, r.grp, q, (const int*)nullptr, r.per_chunks);
    hipLaunchKernelGGL((ns_split_kernel<0>), dim3(4 * r.n_full), dim3(256), 0, stream, r.grp, q, (const int*)nullptr, r.per_full);
  }
  MADIFF_CHECK_LAUNCH();
  NsProduct last = {};
  last.dst = dst;
  return ns_iterate(r, steps, a, b, c, dtype == MADIFF_BF16 ? NS_OUT_BF16 : NS_OUT_F32, last, stream);
}

// ---- Muon plans: a host blob that is copied to the device as it is
extern "C" int madiff_muon_plan(int n, const long* at, const int* rows, const int* cols, const float* scales, void* plan,
                                long plan_bytes, long* need_bytes) {
  if (n < 1 || !at || !rows || !cols || !need_bytes) return -1;
  long ws = 0, chunks = 0, tri = 0, full = 0, need = 0;
  for (int i = 0; i < n; i++) {
    NsMat m;
    if (!ns_describe(m, at[i], rows[i], cols[i], 1.f, ws)) return -1;
    const long ni = m.sp / NS_PAD;
    chunks += m.parts;
    tri += ni * (ni + 1) / 2;
    full += ni * (m.lp / NS_PAD);
    const long end = m.at + (long)m.rows * m.cols;
    need = end > need ? end : need;
    if (chunks > 0x10000000L || tri > 0x10000000L || full > 0x10000000L) return -1;
  }
  NsPlan h = {};
  h.magic = NS_MAGIC;
  h.ws_bytes = ws;
  h.need = need;
  h.mats = n;
  h.chunks = (int)chunks;
  h.tri = (int)tri;
  h.full = (int)full;
  h.at_mats = 256;
  h.at_chunks = h.at_mats + (long)n * sizeof(NsMat);
  h.at_gram = (h.at_chunks + chunks * 8 + 15) / 16 * 16;
  h.at_square = h.at_gram + tri * 16;
  h.at_full = h.at_square + tri * 16;
  h.bytes = h.at_full + full * 16;
  *need_bytes = h.bytes;
  if (!plan) return 0;
  if (plan_bytes < h.bytes) return -1;
  unsigned char* out = (unsigned char*)plan;
  *(NsPlan*)out = h;
  NsMat* mats = (NsMat*)(out + h.at_mats);
  int* ck = (int*)(out + h.at_chunks);
  ws = 0;
  for (int i = 0; i < n; i++) {
    ns_describe(mats[i], at[i], rows[i], cols[i], scales ? scales[i] : 1.f, ws);
    for (int p = 0; p < mats[i].parts; p++) { *ck++ = i; *ck++ = p; }
  }
  int* lists[3] = {(int*)(out + h.at_gram), (int*)(out + h.at_square), (int*)(out + h.at_full)};
  // the tiles with the longest reduction first: they are the last to finish when they start last
  for (int w = 0; w < 3; w++) {
    int* o = lists[w];
    long bound = -1;                                          // lengths in falling order, matrices in the given order
    for (;;) {
      long next = -1;
      for (int i = 0; i < n; i++) {
        const long k = w == 0 ? mats[i].lp : mats[i].sp;
        if ((bound < 0 || k < bound) && k > next) next = k;
      }
      if (next < 0) break;
      for (int i = 0; i < n; i++) {
        const NsMat& m = mats[i];
        if ((w == 0 ? m.lp : m.sp) != next) continue;
        const int ni = m.sp / NS_PAD, nj = m.lp / NS_PAD;
        for (int ti = 0; ti < ni; ti++)
          for (int tj = w == 2 ? 0 : ti; tj < (w == 2 ? nj : ni); tj++) { *o++ = i; *o++ = ti; *o++ = tj; *o++ = 0; }
      }
      bound = next;
    }
  }
  return 0;
}

extern "C" int madiff_muon_plan_ws(const void* plan, long* ws_bytes, long* need_elements) {
  const NsPlan* h = (const NsPlan*)plan;
  if (!h || !ws_bytes || !need_elements || h->magic != NS_MAGIC) return -1;
  *ws_bytes = h->ws_bytes;
  *need_elements = h->need;
  return 0;
}

extern "C" int madiff_muon_step(const void* plan, const void* plan_device, float* p, float* g, float* m, float* ema,
                                void* shadow_bf16, long n, float lr, float momentum, float momentum_rest, int nesterov, float decay,
                                float grad_scale, int zero_grad, int do_ema, float ema_beta, float ema_rest, const int* state,
                                int steps, float a, float b, float c, float eps, void* ws, long ws_bytes, hipStream_t stream) {
  const NsPlan* h = (const NsPlan*)plan;
  if (!h || h->magic != NS_MAGIC || !plan_device || !p || !g || !m || n < h->need || !ws || ws_bytes < h->ws_bytes ||
      ((size_t)ws & 255) || madiff_ortho_check(steps, a, b, c, eps) || do_ema < 0 || do_ema > 2 || (!ema && (do_ema && !state)) ||
      !(momentum >= 0.f && momentum < 1.f))
    return -1;
  const unsigned char* dev = (const unsigned char*)plan_device;
  NsRun r = {};
  r.grp.mats = (const NsMat*)(dev + h->at_mats);
  r.grp.ws = (unsigned char*)ws;
  r.chunks = (const int*)(dev + h->at_chunks);
  r.gram = (const int*)(dev + h->at_gram);
  r.square = (const int*)(dev + h->at_square);
  r.full = (const int*)(dev + h->at_full);
  r.n_chunks = h->chunks;
  r.n_tri = h->tri;
  r.n_full = h->full;
  NsSource q = {};
  q.g = g;
  q.m = m;
  q.mu = momentum;
  q.rest = momentum_rest;
  q.grad_scale = grad_scale;
  q.nesterov = nesterov;
  q.zero_grad = zero_grad;
  q.eps = eps;
  hipLaunchKernelGGL((ns_norm_kernel<2>), dim3(r.n_chunks), dim3(256), 0, stream, r.grp, q, r.chunks, 1);
  hipLaunchKernelGGL((ns_split_kernel<2>), dim3(4 * r.n_full), dim3(256), 0, stream, r.grp, q, r.full, 1);
  MADIFF_CHECK_LAUNCH();
  NsProduct last = {};
  last.p = p;
  last.ema = ema;
  last.shadow = (bf16_t*)shadow_bf16;
  last.decay = decay;
  last.lr = lr;
  last.ema_beta = ema_beta;
  last.ema_rest = ema_rest;
  last.do_ema = do_ema;
  last.state = ema ? state : nullptr;
  return ns_iterate(r, steps, a, b, c, NS_OUT_MUON, last, stream);
}
