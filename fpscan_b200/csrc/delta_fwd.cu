// Gated delta rule, forward over a sequence in chunks of 64 tokens (sm_100a).
// The mathematics and the number format of the products are in delta.cuh.
//
//   delta_prep_kernel   one CTA per (chunk, head), all in parallel: the
//                       64 x 64 matrices N and PN = P N, the decay vectors,
//                       and K and Q as bf16 parts, all in the layout of the
//                       tiles in shared memory.
//   delta_scan_kernel   runs along the chunks of a head: the only sequential
//                       part.
//
// The scan takes 2 C = 32 or 64 values (columns of the state, which never mix)
// per CTA and three products per chunk on tcgen05, each of 128 rows:
//     [K; Q] S0^T         -> X (64 tokens) and Q S0^T (64 tokens),
//     [N; PN] (V - exp(G) X)  -> E and P E, since O's second term is P N R,
//     K^T (beta exp(G_C - G) E)  -> the sum that joins the state,
// so the output costs no product of its own in the chain.  Between them the
// warps read the result from tensor memory (a thread holds C values of one
// token, or of one row of the state), and write the next operand's parts to
// shared memory: warps of lanes 0..63 work on X and E, those of 64..127 on the
// output, all on the state.  What bounds it is this chain, 4500 to 6000 cycles
// a chunk, about 40% of them products, and with 64 heads or more the bytes.
// Measured, dk = dv = 128: two prompts of 8192, 16 heads, bf16 with states 340
// us; 4 x 4096 tokens of 16 heads, bf16 198 us, and 243 us kept for the
// backward pass (1 GB, 4 TB/s).
#include <algorithm>

#include "delta.cuh"
#include "internal.h"

namespace fpscan {

namespace {

// ------------------------------------------------------------------ per-chunk matrices
struct PrepParams {
  const void* q;
  const void* k;
  __nv_bfloat16* kq_tiles;  // [key head][chunk][NP][half of dk][K: 64, Q: 64 rows][64]
  const void* log_decay;
  const void* beta;
  __nv_bfloat16* npn;       // [head][chunk][NS][N: 64, PN: 64 rows][64]
  float* vecs;
  int64_t L, chunks;
  int key_heads, heads, dk;
  float scale;
  int64_t nb;  // sequences (bounds checks of debug builds)
};

// One chunk per CTA of four warps, four CTAs on an SM: a chunk is a chain of
// short steps (load, two 64 x 64 x 128 products, the inverse by blocks of 16,
// P N) with a barrier after each, and what one CTA waits for the others
// cover (with fewer CTAs on an SM 153 us against 128).  4 x 4096 tokens of 16
// heads, dk = 128: bf16 133 us (400 MB, 3 TB/s), 2 x 8192 with three parts 167
// us.  Giving the long rows to another warp in every CTA was no faster.
constexpr int kPrepThreads = 128;
constexpr int kPad = kChunk + 4;  // fp32 rows in shared memory: 16-byte vectors on distinct banks

constexpr int kDkp = 128;                          // dk, padded

// K and Q, and behind them M diag(beta); over K and Q, once they are used up,
// the inverse; behind that, over all else, the images of N and PN.
template <int NP, int NS>
struct PrepCfg {
  static constexpr int kF32 = kChunk * kPad * 4;
  static constexpr int oA = NP * kTileKQ, oImg = kF32;
  static constexpr int kImgEnd = oImg + 2 * NS * kMatBytes;
  static constexpr int oVec = oA + kF32 > kImgEnd ? oA + kF32 : kImgEnd;
  static constexpr int kSmem = oVec + kVecCount * kChunk * 4 + 128;
  static_assert(oImg % 128 == 0);
};

// Where unit u (8 columns) of row r of K (rows 64..: Q) lies in a part.
__device__ __forceinline__ uint32_t kq_at(uint32_t base, int r, int u) {
  return tile_at<128>(base + (u >> 3) * kHalfTile, r, u & 7);
}

// The chunk's rows of x as parts, from row r0 of the tile on.
template <typename T, int NP>
__device__ __forceinline__ void split_tile(uint32_t dst, int r0, const T* x, int64_t stride,
                                           int rows, int units, int tid
                                           FPSCAN_DEBUG_ONLY(, const void* base, int64_t total)) {
  constexpr int U = kDkp / 8, N = kChunk * U / kPrepThreads, V = Elem<T>::kVec;
  if constexpr (NP == 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (tid + i * kPrepThreads) / U, u = (tid + i * kPrepThreads) % U;
      const bool in = r < rows && u < units FPSCAN_DEBUG_ONLY(&& within<T>(x + r * stride + u * 8, 8, base, total));
      cp16(kq_at(dst, r0 + r, u), in ? x + r * stride + u * 8 : x, in);
    }
  } else {
    uint4 raw[N][8 / V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (tid + i * kPrepThreads) / U, u = (tid + i * kPrepThreads) % U;
#pragma unroll
      for (int j = 0; j < 8 / V; ++j)
        raw[i][j] = r < rows && u < units FPSCAN_DEBUG_ONLY(
                                              && within<T>(x + r * stride + u * 8 + j * V, V, base, total))
                        ? *reinterpret_cast<const uint4*>(x + r * stride + u * 8 + j * V)
                        : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (tid + i * kPrepThreads) / U, u = (tid + i * kPrepThreads) % U;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8 / V; ++j) {
        Vec16<T> w;
        w.raw = raw[i][j];
#pragma unroll
        for (int c = 0; c < V; ++c) v[j * V + c] = Elem<T>::load(w.e[c]);
      }
      uint32_t w[4][NP];
#pragma unroll
      for (int c = 0; c < 4; ++c) split_pair<NP>(v[2 * c], v[2 * c + 1], w[c]);
#pragma unroll
      for (int q = 0; q < NP; ++q)
        sts128(kq_at(dst + q * kTileKQ, r0 + r, u), make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]));
    }
  }
}

template <typename T, int NP, int LV>
__global__ void __launch_bounds__(kPrepThreads, 4) delta_prep_kernel(const PrepParams p) {
  constexpr int NS = LV + 1;
  using Cfg = PrepCfg<NP, NS>;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t s_kq = smem_addr(dsm);
  const uint32_t s_img = s_kq + Cfg::oImg;
  float* s_n = reinterpret_cast<float*>(dsm);              // the inverse
  float* s_a = reinterpret_cast<float*>(dsm + Cfg::oA);  // M diag(beta), strictly lower
  float* s_vec = reinterpret_cast<float*>(dsm + Cfg::oVec);
  __shared__ int s_bad;  // first row of M that is not finite

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_bad = kChunk;
  const int64_t bh = blockIdx.x / p.chunks, chunk = blockIdx.x - bh * p.chunks;
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int64_t t0 = chunk * kChunk;
  const int rows = (int)min((int64_t)kChunk, p.L - t0);

  pdl_wait();
  pdl_launch_dependents();
  const int64_t tok_stride = (int64_t)p.key_heads * p.dk;
  const int64_t first = (b * p.L + t0) * tok_stride + (int64_t)hk * p.dk;
  split_tile<T, NP>(s_kq, 0, static_cast<const T*>(p.k) + first, tok_stride, rows, p.dk / 8, tid
                    FPSCAN_DEBUG_ONLY(, p.k, p.nb * p.L * tok_stride));
  split_tile<T, NP>(s_kq, kChunk, static_cast<const T*>(p.q) + first, tok_stride, rows, p.dk / 8, tid
                    FPSCAN_DEBUG_ONLY(, p.q, p.nb * p.L * tok_stride));
  cp_commit();

  // decay vectors: one warp, two tokens a lane; the running sum in 64 bits
  if (warp == 0) {
    const T* g = static_cast<const T*>(p.log_decay) + (b * p.L + t0) * p.heads + h;
    const T* bt = static_cast<const T*>(p.beta) + (b * p.L + t0) * p.heads + h;
    double x[2];
    float be[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = 2 * lane + j;
      FPSCAN_DEBUG_ONLY(const int64_t n_dec = p.nb * p.L * p.heads;
                        if (t < rows && (!within<T, sizeof(T)>(g + (int64_t)t * p.heads, 1, p.log_decay, n_dec) ||
                                         !within<T, sizeof(T)>(bt + (int64_t)t * p.heads, 1, p.beta, n_dec))) continue;)
      float v = t < rows ? Elem<T>::load(g[(int64_t)t * p.heads]) : 0.f;
      if (v < kDecayFloor) v = kDecayFloor;  // NaN stays NaN
      x[j] = v;
      be[j] = t < rows ? Elem<T>::load(bt[(int64_t)t * p.heads]) : 0.f;
    }
    double sum = x[0] + x[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const double cum[2] = {sum - x[1], sum};
    const double all = __shfl_sync(0xffffffffu, sum, 31);
    float* out = p.vecs + (bh * p.chunks + chunk) * (kVecCount * kChunk);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = 2 * lane + j;
      const float hi = (float)cum[j];
      const float v[kVecCount] = {expf((float)cum[j]), expf((float)(all - cum[j])), be[j], hi,
                                  (float)(cum[j] - (double)hi)};
#pragma unroll
      for (int q = 0; q < kVecCount; ++q) {
        s_vec[q * kChunk + t] = v[q];
        FPSCAN_DEBUG_ONLY(if (within<float, 4>(out + q * kChunk + t, 1, p.vecs,
                                               p.nb * p.heads * p.chunks * (kVecCount * kChunk))))
        out[q * kChunk + t] = v[q];
      }
    }
  }
  cp_wait<0>();
  fence_async();
  __syncthreads();
  // the first of the heads that share them keeps the tiles
  const bool keeper = tid == 0 && h % (p.heads / p.key_heads) == 0;
  if (keeper) {
    const int64_t tile = ((b * p.key_heads + hk) * p.chunks + chunk) * NP * (kTileKQ / 2);
    FPSCAN_DEBUG_ONLY(if (within<char>(p.kq_tiles + tile, NP * kTileKQ, p.kq_tiles,
                                       p.nb * p.key_heads * p.chunks * NP * kTileKQ)))
    bulk_s2g(p.kq_tiles + tile, s_kq, NP * kTileKQ);
    bulk_commit();
  }

  // K K^T, then Q K^T, 16 rows a warp; tiles above the diagonal are not needed
  const int g4 = lane >> 2, t4 = lane & 3;
  const float* hi = s_vec + kVecCumHi * kChunk;
  const float* lo = s_vec + kVecCumLo * kChunk;
  const float* be = s_vec + kVecBeta * kChunk;
  const int ksteps = (p.dk + 15) / 16;
  auto with_k = [&](int r0, float (&acc)[8][4]) {  // rows r0.. of the tile times K's
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
#pragma unroll 2
    for (int kk = 0; kk < ksteps; ++kk) {
      const uint32_t half = s_kq + (kk >> 2) * kHalfTile;
      uint32_t af[NP][4];
#pragma unroll
      for (int i = 0; i < NP; ++i)
        ldsm4(af[i], at_a<128>(half + i * kTileKQ, lane, r0 + warp * 16, kk & 3));
#pragma unroll
      for (int np2 = 0; np2 < 4; ++np2) {
        if (np2 > warp) break;
        Step<LV == 2, 2> s;
#pragma unroll
        for (int j = NP - 1; j >= 0; --j) {
          uint32_t bf[4];
          ldsm4(bf, at_b<128>(half + j * kTileKQ, lane, np2 * 16, kk & 3));
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            if (i + j > LV) continue;
            s.mma(0, acc[2 * np2], af[i], bf[0], bf[1]);
            s.mma(1, acc[2 * np2 + 1], af[i], bf[2], bf[3]);
          }
        }
        s.add(0, acc[2 * np2]);
        s.add(1, acc[2 * np2 + 1]);
      }
    }
  };
  float acc[8][4];
  with_k(0, acc);
  // D; with 16-bit results a fast exponential will do (off by 2^-16 at the
  // most where D is above e^-80)
  auto decay = [&](int i, int j) {
    const float x = (hi[i] - hi[j]) + (lo[i] - lo[j]);
    return LV == 1 ? __expf(x) : expf(x);
  };
  float probe[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    if (n > 2 * warp + 1) break;  // above the diagonal, and not read
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = warp * 16 + g4 + r * 8, j0 = n * 8 + 2 * t4;
      float a[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j = j0 + c;
        a[c] = i > j ? acc[n][2 * r + c] * decay(i, j) * be[j] : 0.f;
        probe[r] = fmaf(a[c], 0.f, probe[r]);
      }
      *reinterpret_cast<float2*>(&s_a[i * kPad + j0]) = make_float2(a[0], a[1]);
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r)
    if (probe[r] != 0.f) atomicMin(&s_bad, warp * 16 + g4 + r * 8);
  with_k(kChunk, acc);
  if (keeper) bulk_wait_read<0>();
  __syncthreads();  // K and Q are used up
  // An infinity or a NaN (of k, beta, log_decay; or an overflow) would reach
  // the rows of N before its own through zeros times it.  From that row on M
  // counts as zeros here, and what reads the state as NaN, which
  // delta_scan_kernel carries to all that follows.
  if (s_bad < kChunk) {  // uniform
    for (int i = s_bad * kPad + tid; i < kChunk * kPad; i += kPrepThreads) s_a[i] = 0.f;
    for (int i = s_bad + tid; i < kChunk; i += kPrepThreads)
      FPSCAN_DEBUG_ONLY(if (within<float, 4>(p.vecs + (bh * p.chunks + chunk) * (kVecCount * kChunk) + kVecEnter * kChunk + i,
                                             1, p.vecs, p.nb * p.heads * p.chunks * (kVecCount * kChunk))))
      p.vecs[(bh * p.chunks + chunk) * (kVecCount * kChunk) + kVecEnter * kChunk + i] =
          __int_as_float(0x7fc00000);
    __syncthreads();
  }
  uint32_t pf[4][NS][4];  // P's 16 rows of this warp, as an A operand
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (kk > warp) break;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = 2 * kk + (q >> 1), r = q & 1;
      const int i = warp * 16 + g4 + r * 8, j0 = n * 8 + 2 * t4;
      float v[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j = j0 + c;
        const float d = i > j ? decay(i, j) : 1.f;
        v[c] = i >= j ? acc[n][2 * r + c] * d * p.scale * be[j] : 0.f;
      }
      uint32_t w[NS];
      split_pair<NS>(v[0], v[1], w);
#pragma unroll
      for (int o = 0; o < NS; ++o) pf[kk][o][q] = w[o];
    }
  }

  // N = (I + A)^-1.  16 x 16 blocks on the diagonal by substitution, a column
  // a lane; then [[B, 0], [C, D]]^-1 = [[B', 0], [-D' C B', D']] twice.
  {
    const int o = warp * 16;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == (lane & 15) ? 1.f : 0.f;
      const float4* a = reinterpret_cast<const float4*>(&s_a[(o + i) * kPad + o]);
#pragma unroll
      for (int l4 = 0; l4 < (i + 3) / 4; ++l4) {
        const float4 q = a[l4];
        if (4 * l4 < i) v = fmaf(-q.x, x[4 * l4], v);
        if (4 * l4 + 1 < i) v = fmaf(-q.y, x[4 * l4 + 1], v);
        if (4 * l4 + 2 < i) v = fmaf(-q.z, x[4 * l4 + 2], v);
        if (4 * l4 + 3 < i) v = fmaf(-q.w, x[4 * l4 + 3], v);
      }
      x[i] = v;
    }
    // lanes 0..15 store the block; 16..31 clear the block to its right
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int col = o + lane;
      if (col < kChunk) s_n[(o + i) * kPad + col] = lane < 16 ? x[i] : 0.f;
    }
    for (int i = 0; i < 16; ++i)  // and the blocks beyond
      for (int col = o + 32 + lane; col < kChunk; col += 32) s_n[(o + i) * kPad + col] = 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int half = 16; half <= 32; half <<= 1) {
    // per 2*half block: rows half..2*half, columns 0..half.  A thread takes 2
    // rows x 4 columns; 16-byte vectors along both.
    const int per = half * half / 8;  // threads of a block: 32, 128
    const int blk = tid / per, in = tid % per;
    const bool on = blk < 32 / half;
    const int col = in % (half / 4) * 4, row = in / (half / 4) * 2;
    const int o = blk * 2 * half;
    float4 r0, r1;
    auto product = [&](const float* left, const float* right, int lo_, int ro) {
      // rows row, row + 1 of left (columns lo_..) x rows of right (columns ro + col..)
      r0 = r1 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int l = 0; l < half; l += 4) {
        const float4 a0 = *reinterpret_cast<const float4*>(&left[(o + half + row) * kPad + lo_ + l]);
        const float4 a1 = *reinterpret_cast<const float4*>(&left[(o + half + row + 1) * kPad + lo_ + l]);
        const float x0[4] = {a0.x, a0.y, a0.z, a0.w}, x1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4 y = *reinterpret_cast<const float4*>(&right[(ro + l + q) * kPad + o + col]);
          r0.x = fmaf(x0[q], y.x, r0.x);
          r0.y = fmaf(x0[q], y.y, r0.y);
          r0.z = fmaf(x0[q], y.z, r0.z);
          r0.w = fmaf(x0[q], y.w, r0.w);
          r1.x = fmaf(x1[q], y.x, r1.x);
          r1.y = fmaf(x1[q], y.y, r1.y);
          r1.z = fmaf(x1[q], y.z, r1.z);
          r1.w = fmaf(x1[q], y.w, r1.w);
        }
      }
    };
    // C B' over C, then -D' (C B') into the inverse
    if (on) product(s_a, s_n, o, o);
    __syncthreads();
    if (on) {
      *reinterpret_cast<float4*>(&s_a[(o + half + row) * kPad + o + col]) = r0;
      *reinterpret_cast<float4*>(&s_a[(o + half + row + 1) * kPad + o + col]) = r1;
    }
    __syncthreads();
    if (on) {
      product(s_n, s_a, o + half, o + half);
      *reinterpret_cast<float4*>(&s_n[(o + half + row) * kPad + o + col]) =
          make_float4(-r0.x, -r0.y, -r0.z, -r0.w);
      *reinterpret_cast<float4*>(&s_n[(o + half + row + 1) * kPad + o + col]) =
          make_float4(-r1.x, -r1.y, -r1.z, -r1.w);
    }
    __syncthreads();
  }

  // N's image, then PN's: rows 64.. of the same tile
  for (int s = tid; s < kChunk * kChunk / 8; s += kPrepThreads) {
    const int i = s / (kChunk / 8), j0 = (s % (kChunk / 8)) * 8;
    const float4 x = *reinterpret_cast<const float4*>(&s_n[i * kPad + j0]);
    const float4 y = *reinterpret_cast<const float4*>(&s_n[i * kPad + j0 + 4]);
    uint32_t w[4][NS];
    split_pair<NS>(x.x, x.y, w[0]);
    split_pair<NS>(x.z, x.w, w[1]);
    split_pair<NS>(y.x, y.y, w[2]);
    split_pair<NS>(y.z, y.w, w[3]);
#pragma unroll
    for (int q = 0; q < NS; ++q)
      sts128(tile_at<128>(s_img + 2 * q * kMatBytes, i, j0 / 8),
             make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]));
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    if (kk > warp) break;
#pragma unroll
    for (int n2 = 0; n2 <= kk; ++n2) {
      Step<LV == 2, 2> s;
#pragma unroll
      for (int j = LV; j >= 0; --j) {
        uint32_t nb[4];
        ldsm4_t(nb, at_bt<128>(s_img + 2 * j * kMatBytes, lane, n2 * 16, kk));
#pragma unroll
        for (int i = LV - j; i >= 0; --i) {
          s.mma(0, acc[2 * n2], pf[kk][i], nb[0], nb[1]);
          s.mma(1, acc[2 * n2 + 1], pf[kk][i], nb[2], nb[3]);
        }
      }
      s.add(0, acc[2 * n2]);
      s.add(1, acc[2 * n2 + 1]);
    }
  }
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    uint32_t a[NS][4];
    split_frag<NS>(acc[2 * kk], acc[2 * kk + 1], a);
#pragma unroll
    for (int q = 0; q < NS; ++q)
      stsm4(at_a<128>(s_img + 2 * q * kMatBytes, lane, kChunk + warp * 16, kk), a[q]);
  }
  fence_async();
  __syncthreads();
  if (tid == 0) {
    FPSCAN_DEBUG_ONLY(if (within<char>(p.npn + (bh * p.chunks + chunk) * NS * (2 * kChunk * kChunk), 2 * NS * kMatBytes,
                                       p.npn, p.nb * p.heads * p.chunks * 2 * NS * kMatBytes)))
    bulk_s2g(p.npn + (bh * p.chunks + chunk) * NS * (2 * kChunk * kChunk), s_img, 2 * NS * kMatBytes);
    bulk_commit();
    bulk_wait_all();
  }
}

// ------------------------------------------------------------------ along the chunks
struct ScanParams {
  const __nv_bfloat16* kq_tiles;
  const void* v;
  const __nv_bfloat16* npn;
  const float* vecs;
  const float* initial;
  float* final_state;
  void* out;                  // KEEP false
  __nv_bfloat16* e_parts;     // KEEP true: strips [head][chunk][dv / 16][NS][64][16]
  __nv_bfloat16* s_parts;     //                   [head][chunk][dv / 16][NS][128][16]
  int64_t L, chunks;
  int key_heads, heads, dk, dv, slices;
  float scale;
  int64_t nb;  // sequences (bounds checks of debug builds)
};

constexpr int kScanThreads = 256;

template <typename T, int LV, int C>
struct ScanCfg {
  static constexpr int NP = kParts<T>;
  static constexpr int NS = LV + 1;
  static constexpr int kKQ = NP * kTileKQ;
  static constexpr int kNPN = NS * 2 * kMatBytes;
  static constexpr int kPartS = 128 * 4 * C, kPartE = kChunk * 4 * C;  // of S0; of R and E
  static constexpr int kVec = 3 * kChunk * 4;                      // enter, leave, beta
  static constexpr int kFixed = kNPN + NS * kPartS + NS * kPartE + NextRow<T, C>::kBytes;
  static constexpr int kRoom = 227 * 1024 - 2 * 1024;  // alignment; static
  static constexpr int kSt = kFixed + 2 * (kKQ + kVec) <= kRoom ? 2 : 1;  // stages of K, Q
  static constexpr int oNPN = kSt * kKQ, oS = oNPN + kNPN, oE = oS + NS * kPartS;
  static constexpr int oRow = oE + NS * kPartE, oVec = oRow + NextRow<T, C>::kBytes;
  static constexpr int kSmem = oVec + kSt * kVec + 1024;
  static_assert(kSmem + 1024 <= 227 * 1024);
};

// KEEP: no output; E and the states entering the chunks are written as parts
// (what the backward pass multiplies with).
template <typename T, int LV, bool KEEP, int C>
__global__ void __launch_bounds__(kScanThreads, 1) delta_scan_kernel(const ScanParams p) {
  using Cfg = ScanCfg<T, LV, C>;
  constexpr int kTmem = kTmemColumns<LV, C>;
  constexpr int NP = Cfg::NP, NS = Cfg::NS;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sm0 = smem_addr(dsm);
  const uint32_t s_npn = sm0 + Cfg::oNPN, s_s = sm0 + Cfg::oS, s_e = sm0 + Cfg::oE;
  __shared__ __align__(8) uint64_t full_kq[2], full_n, done[3];
  __shared__ uint32_t s_tmem;
  __shared__ int s_bad[2], s_first[2 * C];  // see `bad` below

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform
  const int quad = warp & 3, col0 = (warp >> 2) * C;  // tensor memory lanes 32 quad.., columns
  const bool is_x = quad < 2;                          // X and E; else the output
  const int tok = (quad & 1) * 32 + lane;              // this thread's token
  const int dk = quad * 32 + lane;                     // and row of the state
  const int64_t bh = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - bh * p.slices);
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int dv0 = slice * 2 * C + col0;
  const int nval = min(C, p.dv - dv0);  // values of this thread's C that exist (may be <= 0)
  const int strips = (p.dv + 15) / 16;
  const int64_t vstride = (int64_t)p.heads * p.dv;
  const int64_t tile = (b * p.key_heads + hk) * p.chunks, unit0 = bh * p.chunks;
  FPSCAN_DEBUG_ONLY(const int64_t n_units = p.nb * p.heads * p.chunks, n_tiles = p.nb * p.key_heads * p.chunks,
                    n_v = p.nb * p.L * vstride, n_state = p.nb * p.heads * p.dv * p.dk;)

  if (tid == 0) {
    mbar_init(&full_kq[0], 1);
    mbar_init(&full_kq[1], 1);
    mbar_init(&full_n, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&done[i], 1);
    fence_mbar_init();
    s_bad[0] = s_bad[1] = 0;
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&s_tmem)), "n"(kTmem)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  umma_fence_before();
  __syncthreads();
  umma_fence_after();
  const uint32_t tmem = s_tmem, tmem2 = tmem + NS * 2 * C;  // first and third product; second
  const uint32_t my_tmem = tmem + ((uint32_t)(quad * 32) << 16) + col0;
  pdl_wait();
  pdl_launch_dependents();

  // Copies are issued by an elected lane of a converged warp (a lone thread of
  // a divergent branch takes over 100 cycles for each).
  const bool loads = warp == kScanThreads / 32 - 1;
  auto load_kq = [&](int64_t c) {
    __syncwarp();
    const int s = (int)(c % Cfg::kSt);
    if (elect_one()) {
      mbar_expect_tx(&full_kq[s], Cfg::kKQ + Cfg::kVec);
      // (a copy left out: the wait for it gives up and is recorded too)
      FPSCAN_DEBUG_ONLY(if (within<char>(p.kq_tiles + (tile + c) * (Cfg::kKQ / 2), Cfg::kKQ, p.kq_tiles, n_tiles * Cfg::kKQ) &&
                            within<float>(p.vecs + (unit0 + c) * (kVecCount * kChunk), Cfg::kVec / 4, p.vecs,
                                          n_units * (kVecCount * kChunk))) {)
      bulk_in(sm0 + s * Cfg::kKQ, p.kq_tiles + (tile + c) * (Cfg::kKQ / 2), Cfg::kKQ, &full_kq[s]);
      bulk_in(sm0 + Cfg::oVec + s * Cfg::kVec, p.vecs + (unit0 + c) * (kVecCount * kChunk), Cfg::kVec,
              &full_kq[s]);
      FPSCAN_DEBUG_ONLY(})
    }
    __syncwarp();
  };
  auto load_n = [&](int64_t c) {
    __syncwarp();
    if (elect_one()) {
      mbar_expect_tx(&full_n, Cfg::kNPN);
      FPSCAN_DEBUG_ONLY(if (within<char>(p.npn + (unit0 + c) * (Cfg::kNPN / 2), Cfg::kNPN, p.npn, n_units * Cfg::kNPN)))
      bulk_in(s_npn, p.npn + (unit0 + c) * (Cfg::kNPN / 2), Cfg::kNPN, &full_n);
    }
    __syncwarp();
  };
  if (loads) {
    for (int64_t c = 0; c < min((int64_t)Cfg::kSt, p.chunks); ++c) load_kq(c);
    load_n(0);
  }

  const T* v_row = static_cast<const T*>(p.v) + (b * p.L + tok) * vstride + (int64_t)h * p.dv + dv0;
  NextRow<T, C> v_next(sm0 + Cfg::oRow, (warp >> 2) * 64 + tok);
  if (is_x) v_next.fetch(v_row, tok < p.L ? nval : 0, static_cast<const T*>(p.v) FPSCAN_DEBUG_ONLY(, n_v));

  float S[C];
#pragma unroll
  for (int i = 0; i < C; ++i)
    S[i] = p.initial != nullptr && dk < p.dk && i < nval FPSCAN_DEBUG_ONLY(
               && within<float, 4>(p.initial + (bh * p.dv + dv0 + i) * p.dk + dk, 1, p.initial, n_state))
               ? p.initial[(bh * p.dv + dv0 + i) * p.dk + dk]
               : 0.f;
  const int ksteps = (p.dk + 15) / 16;
  const float nan = __int_as_float(0x7fc00000);

  // A wait that gave up is recorded; later waits are skipped, and every thread
  // still meets every barrier.
  bool ok = true;
  auto wait = [&](uint64_t* bar, int64_t phase) {
    if (ok) ok = mbar_wait_soon(bar, (uint32_t)(phase & 1));
  };
  for (int64_t c = 0; c < p.chunks; ++c) {
    const int s = (int)(c % Cfg::kSt);
    const uint32_t s_kq = sm0 + s * Cfg::kKQ;
    const float* vec = reinterpret_cast<const float*>(dsm + Cfg::oVec + s * Cfg::kVec);

    // S0's parts, rows of dk
    split_row<NS>(S, [&](int q, int u, const uint4& w) {
      sts128(val_at<C>(s_s + q * Cfg::kPartS, dk, col0 / 8 + u), w);
    });
    fence_async();
    umma_fence_before();
    __syncthreads();
    // every thread is through with the chunk before
    if (loads && c > 0 && c + Cfg::kSt - 1 < p.chunks) load_kq(c + Cfg::kSt - 1);
    if (tid == 0) s_bad[(c + 1) & 1] = 0;
    if (warp == 0) {
      umma_fence_after();
      wait(&full_kq[s], c / Cfg::kSt);
      if (elect_one()) {
        umma_parts<C, NP, LV, kDkp / 16, true, false>(tmem, umma_desc_a(s_kq, 16),
                                                      umma_desc_b<C>(s_s, Cfg::kPartS), kTileKQ, 32, 64 * C,
                                                      kHalfTile, ksteps);
        umma_commit(&done[0]);
      }
      __syncwarp();
    }
    if (KEEP)  // S0's parts to their strips, from the registers, while the product runs
      split_row<NS>(S, [&](int q, int u, const uint4& w) {
        if ((u & ~1) * 8 < nval) {
          char* sp = reinterpret_cast<char*>(p.s_parts) +
                     (((unit0 + c) * strips + dv0 / 16 + (u >> 1)) * NS + q) * (int64_t)(2 * kStrip) +
                     strip_at(0, dk, u & 1);
          FPSCAN_DEBUG_ONLY(if (within<char>(sp, 16, p.s_parts, n_units * strips * NS * 2 * kStrip)))
          *reinterpret_cast<uint4*>(sp) = w;
        }
      });
    wait(&full_kq[s], c / Cfg::kSt);  // the vectors
    const float ge = vec[kVecEnter * kChunk + tok], total = vec[kVecEnter * kChunk + kChunk - 1];
    const float wb = vec[kVecLeave * kChunk + tok] * vec[kVecBeta * kChunk + tok];
    wait(&done[0], c);
    umma_fence_after();

    float x[C];
    tmem_sum<NS>(my_tmem, x);
    // An infinity or a NaN in R (of v, k, or the state) spoils its value from
    // that token on, but the zeros above the diagonals of N and PN would carry
    // it to earlier tokens: it is taken out here and put back into E, O and
    // the state afterwards (s_first: first such token of each value).
    if (is_x) {
      float probe[4] = {0.f, 0.f, 0.f, 0.f};
      float v[C];
      v_next.take(v);
#pragma unroll
      for (int i = 0; i < C; ++i) {
        x[i] = fmaf(-ge, x[i], v[i]);
        probe[i & 3] = fmaf(x[i], 0.f, probe[i & 3]);
      }
      if ((probe[0] + probe[1]) + (probe[2] + probe[3]) != 0.f) s_bad[c & 1] = 1;
      split_row<NS>(x, [&](int q, int u, const uint4& w) {
        sts128(val_at<C>(s_e + q * Cfg::kPartE, tok, col0 / 8 + u), w);
      });
      fence_async();
      // v of the next chunk
      if (c + 1 < p.chunks) {
        v_row += kChunk * vstride;
        v_next.fetch(v_row, (c + 1) * kChunk + tok < p.L ? nval : 0,
                     static_cast<const T*>(p.v) FPSCAN_DEBUG_ONLY(, n_v));
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) x[i] *= ge * p.scale;
    }
    umma_fence_before();
    __syncthreads();
    const bool bad = s_bad[c & 1] != 0;
    if (bad) {  // uniform
      if (tid < 2 * C) s_first[tid] = kChunk;
      __syncthreads();
      if (is_x)
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (!(fabsf(x[i]) <= 3.38e38f)) atomicMin(&s_first[col0 + i], tok);
      __syncthreads();
      if (is_x) {
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (tok >= s_first[col0 + i]) x[i] = 0.f;
        split_row<NS>(x, [&](int q, int u, const uint4& w) {
          sts128(val_at<C>(s_e + q * Cfg::kPartE, tok, col0 / 8 + u), w);
        });
        fence_async();
      }
      __syncthreads();
    }
    if (warp == 0) {
      umma_fence_after();
      wait(&full_n, c);
      if (elect_one()) {
        umma_parts<C, NS, LV, kChunk / 16, false, false>(tmem2, umma_desc_a(s_npn, 16),
                                                         umma_desc_b<C>(s_e, Cfg::kPartE), 2 * kMatBytes, 32,
                                                         64 * C, 0, kChunk / 16);
        umma_commit(&done[1]);
      }
      __syncwarp();
    }
    wait(&done[1], c);
    umma_fence_after();
    if (loads && c + 1 < p.chunks) load_n(c + 1);  // N and PN are used up

    if (is_x) {
      tmem_sum<NS>(my_tmem + NS * 2 * C, x);
      if (KEEP) {
        if (bad)
#pragma unroll
          for (int i = 0; i < C; ++i)
            if (tok >= s_first[col0 + i]) x[i] = nan;
        split_row<NS>(x, [&](int q, int u, const uint4& w) {
          if ((u & ~1) * 8 < nval) {
            char* ep = reinterpret_cast<char*>(
                p.e_parts +
                (((unit0 + c) * strips + dv0 / 16 + (u >> 1)) * NS + q) * (kStrip / 2));
            FPSCAN_DEBUG_ONLY(if (within<char>(ep + strip_at(0, tok, u & 1), 16, p.e_parts, n_units * strips * NS * kStrip)))
            *reinterpret_cast<uint4*>(ep + strip_at(0, tok, u & 1)) = w;
          }
        });
      }
#pragma unroll
      for (int i = 0; i < C; ++i) x[i] *= wb;
      split_row<NS>(x, [&](int q, int u, const uint4& w) {
        sts128(val_at<C>(s_e + q * Cfg::kPartE, tok, col0 / 8 + u), w);
      });
      fence_async();
      umma_fence_before();
      asm volatile("bar.sync 1, 128;" ::: "memory");  // the warps of X and E
      if (warp == 0) {
        umma_fence_after();
        if (elect_one()) {
          umma_parts<C, NP, LV, kChunk / 16, false, true>(tmem, umma_desc_a(s_kq, kHalfTile),
                                                          umma_desc_b<C>(s_e, Cfg::kPartE), kTileKQ, 2048,
                                                          64 * C, 0, kChunk / 16);
          umma_commit(&done[2]);
        }
        __syncwarp();
      }
    } else if (!KEEP) {
      float pe[C];
      tmem_sum<NS>(my_tmem + NS * 2 * C, pe);
#pragma unroll
      for (int i = 0; i < C; ++i) x[i] += pe[i];
      if (bad)
#pragma unroll
        for (int i = 0; i < C; ++i)
          if (tok >= s_first[col0 + i]) x[i] = nan;
      if (c * kChunk + tok < p.L)
        store_row<T>(static_cast<T*>(p.out) + (b * p.L + c * kChunk + tok) * vstride +
                         (int64_t)h * p.dv + dv0,
                     nval, x FPSCAN_DEBUG_ONLY(, p.out, n_v));
    }
    wait(&done[2], c);
    umma_fence_after();
    // The chunk's sum starts at zero and joins the state in one rounded
    // multiply-add.
    tmem_sum<NS>(my_tmem, x);
#pragma unroll
    for (int i = 0; i < C; ++i) S[i] = fmaf(total, S[i], x[i]);
    if (bad)
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (s_first[col0 + i] < kChunk) S[i] = nan;
  }

  if (!KEEP && p.final_state != nullptr && ok && dk < p.dk)
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (i < nval FPSCAN_DEBUG_ONLY(&& within<float, 4>(p.final_state + (bh * p.dv + dv0 + i) * p.dk + dk, 1,
                                                         p.final_state, n_state)))
        p.final_state[(bh * p.dv + dv0 + i) * p.dk + dk] = S[i];
  // No copy may land after the CTA is gone: at once, unless a wait gave up.
  if (loads) {
    for (int64_t c = max((int64_t)0, p.chunks - Cfg::kSt); c < p.chunks; ++c)
      mbar_wait_soon(&full_kq[c % Cfg::kSt], (uint32_t)((c / Cfg::kSt) & 1));
    mbar_wait_soon(&full_n, (uint32_t)((p.chunks - 1) & 1));
  }
  umma_fence_before();
  __syncthreads();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmem));
}

// ------------------------------------------------------------------ host side
template <typename Kern>
cudaError_t configure(Kern kern, int smem) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
}

template <typename T, int LV, bool KEEP, int C>
cudaError_t launch_scan_as(const DeltaArgs& a, ScanParams& p, int64_t bh) {
  using Cfg = ScanCfg<T, LV, C>;
  auto kern = delta_scan_kernel<T, LV, KEEP, C>;
  const cudaError_t e = configure(kern, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  p.slices = (int)((a.dv + 2 * C - 1) / (2 * C));
  return launch_pdl(kern, (unsigned)(bh * p.slices), kScanThreads, Cfg::kSmem, a.stream, p);
}

// 32 values per CTA while every CTA gets an SM of its own (fewer values,
// shorter steps: two prompts of 8192, 16 heads with states, 340 us against
// 532 us), 64 beyond (more work for each operand read: 4 x 4096 of 16 heads
// 198 us against 280 us, kept for the backward pass 243 us against 300 us,
// delta_rev_kernel 284 us against 325 us).
template <typename T, int LV, bool KEEP>
cudaError_t launch_scan(const DeltaArgs& a, ScanParams& p, int64_t bh) {
  return bh * ((a.dv + 31) / 32) <= a.num_sms ? launch_scan_as<T, LV, KEEP, 16>(a, p, bh)
                                              : launch_scan_as<T, LV, KEEP, 32>(a, p, bh);
}

}  // namespace

// Prep and scan for sequences [b0, b0 + nb) of the call.  keep: for the
// backward pass (E and the states instead of the output).
template <typename T, int LV>
cudaError_t delta_fwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb,
                           bool keep) {
  constexpr int NP = kParts<T>;
  char* ws = static_cast<char*>(a.workspace);
  auto bf = [&](int64_t off) { return reinterpret_cast<__nv_bfloat16*>(ws + off); };
  const int64_t k0 = b0 * a.seqlen * a.key_heads * a.dk, v0 = b0 * a.seqlen * a.heads * a.dv;
  const int64_t g0 = b0 * a.seqlen * a.heads, s0 = b0 * a.heads * a.dv * a.dk;
  const int64_t bh = nb * a.heads;
  PrepParams pp{};
  pp.q = static_cast<const T*>(a.q) + k0;
  pp.k = static_cast<const T*>(a.k) + k0;
  pp.kq_tiles = bf(pl.kq_tiles);
  pp.log_decay = static_cast<const T*>(a.log_decay) + g0;
  pp.beta = static_cast<const T*>(a.beta) + g0;
  pp.npn = bf(pl.npn);
  pp.vecs = reinterpret_cast<float*>(ws + pl.vecs);
  pp.L = a.seqlen;
  pp.chunks = pl.chunks;
  pp.key_heads = (int)a.key_heads;
  pp.heads = (int)a.heads;
  pp.dk = (int)a.dk;
  pp.scale = a.scale;
  pp.nb = nb;
  auto prep = delta_prep_kernel<T, NP, LV>;
  constexpr int prep_smem = PrepCfg<NP, LV + 1>::kSmem;
  cudaError_t e = configure(prep, prep_smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(prep, (unsigned)(bh * pl.chunks), kPrepThreads, prep_smem, a.stream, pp);
  if (e != cudaSuccess) return e;

  ScanParams p{};
  p.kq_tiles = pp.kq_tiles;
  p.v = static_cast<const T*>(a.v) + v0;
  p.npn = pp.npn;
  p.vecs = pp.vecs;
  p.initial = a.initial ? a.initial + s0 : nullptr;
  p.final_state = !keep && a.final_state ? a.final_state + s0 : nullptr;
  p.out = keep ? nullptr : static_cast<T*>(a.out) + v0;
  p.e_parts = bf(pl.e_parts);
  p.s_parts = bf(pl.s_parts);
  p.L = a.seqlen;
  p.chunks = pl.chunks;
  p.key_heads = (int)a.key_heads;
  p.heads = (int)a.heads;
  p.dk = (int)a.dk;
  p.dv = (int)a.dv;
  p.scale = a.scale;
  p.nb = nb;
  return keep ? launch_scan<T, LV, true>(a, p, bh) : launch_scan<T, LV, false>(a, p, bh);
}

template cudaError_t delta_fwd_pass<__nv_bfloat16, 1>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__nv_bfloat16, 2>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__half, 1>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__half, 2>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<float, 2>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);

DeltaPlan delta_plan(int64_t batch, int64_t seqlen, int64_t key_heads, int64_t heads, int64_t dk,
                     int64_t dv, int dtype, bool wide, bool backward) {
  DeltaPlan pl{};
  pl.np = dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1;
  pl.ns = wide || dtype == kF32 ? 3 : 2;
  pl.chunks = (seqlen + kChunk - 1) / kChunk;
  // Sequences per pass: what the passes keep is held to 2 GiB (or one
  // sequence's), so a long batch does not multiply the workspace.
  for (pl.batch = batch;; pl.batch = (pl.batch + 1) / 2) {
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
      const int64_t o = at;
      at += (bytes + 255) / 256 * 256;
      return o;
    };
    const int64_t nb = pl.batch, c = nb * heads * pl.chunks, tok = nb * seqlen;
    pl.kq_tiles = take(nb * key_heads * pl.chunks * pl.np * kTileKQ);
    pl.npn = take(c * pl.ns * 2 * kMatBytes);
    pl.vecs = take(c * kVecCount * kChunk * 4);
    if (backward) {
      const int64_t strips = (dv + 15) / 16;
      pl.do_parts = take(c * pl.np * kStrip * strips);
      pl.e_parts = take(c * pl.ns * kStrip * strips);
      pl.dv_parts = take(c * pl.ns * kStrip * strips);
      pl.s_parts = take(c * pl.ns * 2 * kStrip * strips);
      pl.ds_parts = take(c * pl.ns * 2 * kStrip * strips);
      if (heads != key_heads) {
        pl.dq_part = take(tok * heads * dk * 4);
        pl.dk_part = take(tok * heads * dk * 4);
      }
    }
    pl.bytes = at;
    if (at <= (int64_t(2) << 30) || pl.batch <= 1) return pl;
  }
}

namespace {
template <typename T, int LV>
cudaError_t fwd_all(const DeltaArgs& a, const DeltaPlan& pl) {
  for (int64_t b0 = 0; b0 < a.batch; b0 += pl.batch) {
    const int64_t nb = std::min(pl.batch, a.batch - b0);
    const cudaError_t e = delta_fwd_pass<T, LV>(a, pl, b0, nb, false);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}
}  // namespace

cudaError_t launch_delta_fwd(const DeltaArgs& a) {
  const DeltaPlan pl = delta_plan(a.batch, a.seqlen, a.key_heads, a.heads, a.dk, a.dv, a.dtype,
                                  a.wide != 0, false);
  switch (a.dtype) {
    case kF32:
      return fwd_all<float, 2>(a, pl);
    case kF16:
      return a.wide ? fwd_all<__half, 2>(a, pl) : fwd_all<__half, 1>(a, pl);
    default:
      return a.wide ? fwd_all<__nv_bfloat16, 2>(a, pl) : fwd_all<__nv_bfloat16, 1>(a, pl);
  }
}

}  // namespace fpscan
