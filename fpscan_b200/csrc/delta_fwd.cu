// Gated delta rule, forward over a sequence in chunks of 64 tokens (sm_100a).
// The mathematics and the number format of the products are in delta.cuh.
//
//   delta_prep_kernel   one CTA per (chunk, head), all in parallel: the
//                       64 x 64 matrices N and P, the decay vectors, and K
//                       and Q as bf16 parts in the layout of the tiles in
//                       shared memory.
//   delta_scan_kernel   runs along the chunks of a head with the state in
//                       registers: the only sequential part.
//
// The scan keeps the state transposed, S^T tiles as accumulators: a warp
// owns 16 rows of values (dv) and all of dk (64 registers a thread at
// dk = 128).  Every product of the chain then has the warp's own rows as its
// A operand -- K S0^T, N R, the state's update -- and an accumulator turns
// into the next product's A operand by packing registers, so the chain of a
// chunk needs no barrier between its products.  Columns of the state never
// mix, so a head is cut along dv over as many CTAs as the GPU has room for.
//
// A chunk's products wait for one another, and one warp alone issues only
// about every sixth cycle, so the 16 rows are shared by three warps:
//   two chain warps  each with half of dk: their parts of K S0^T are summed
//                    through shared memory, each computes E for half of the
//                    tokens, and each updates its half of the state;
//   an output warp   O = scale exp(G) Q S0^T + P E, from the parts of S0 and
//                    from E in shared memory, while the chain goes on to the
//                    update and the next chunk.
// K, N (chain) and Q, P (output) come by bulk copies through a ring of one or
// two stages each, issued by the first chain and the first output warp.
// Where the states and E are kept for the backward pass there is no output,
// and one more warp loads.
#include <algorithm>

#include "delta.cuh"
#include "internal.h"

namespace fpscan {

namespace {

// ------------------------------------------------------------------ per-chunk matrices
struct PrepParams {
  const void* q;
  const void* k;
  __nv_bfloat16* q_tiles;   // [key head][chunk][NP][64][DKP], as in shared memory
  __nv_bfloat16* k_tiles;
  const void* log_decay;
  const void* beta;
  __nv_bfloat16* n_mat;
  __nv_bfloat16* p_mat;
  float* vecs;
  int64_t L, chunks;
  int key_heads, heads, dk;
  float scale;
};

constexpr int kPrepThreads = 128;
constexpr int kMatBytes = kChunk * kChunk * 2;  // one part of N or P
constexpr int kPad = kChunk + 4;  // fp32 rows in shared memory: 16-byte vectors on distinct banks

// K and Q; over them, once they are used up, the image of P and the inverse.
template <int NP, int NS, int DKP>
struct PrepCfg {
  static constexpr int kTile = kChunk * DKP * 2;
  static constexpr int kF32 = kChunk * kPad * 4;
  static constexpr int kTiles = 2 * NP * kTile;
  static constexpr int oN = NS * kMatBytes;  // the image of P lies at 0
  static constexpr int kBody = kTiles > oN + kF32 ? kTiles : oN + kF32;
  static constexpr int oA = kBody, oVec = oA + kF32;
  static constexpr int kSmem = oVec + kVecCount * kChunk * 4 + 128;
};

// The chunk's rows of x as parts in a tile: 16-byte units of 8 values.
template <typename T, int NP, int DKP>
__device__ __forceinline__ void split_tile(uint32_t dst, const T* x, int64_t stride, int rows,
                                           int units, int tid) {
  constexpr int ROWB = DKP * 2, U = DKP / 8, N = kChunk * U / kPrepThreads, V = Elem<T>::kVec;
  if constexpr (NP == 1) {
    load_tile<kChunk, ROWB, kPrepThreads>(dst, x, stride * 2, rows, units, tid);
  } else {
    uint4 raw[N][8 / V];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (tid + i * kPrepThreads) / U, u = (tid + i * kPrepThreads) % U;
#pragma unroll
      for (int j = 0; j < 8 / V; ++j)
        raw[i][j] = r < rows && u < units
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
        sts128(tile_at<ROWB>(dst + q * kChunk * ROWB, r, u),
               make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]));
    }
  }
}

template <typename T, int NP, int LV, int DKP>
__global__ void __launch_bounds__(kPrepThreads, 4) delta_prep_kernel(const PrepParams p) {
  constexpr int NS = LV + 1;
  constexpr int ROWB = DKP * 2, TILE = kChunk * ROWB, MROW = kChunk * 2;
  using Cfg = PrepCfg<NP, NS, DKP>;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t s_k = smem_addr(dsm), s_q = s_k + NP * TILE;
  float* s_n = reinterpret_cast<float*>(dsm + Cfg::oN);  // the inverse
  float* s_a = reinterpret_cast<float*>(dsm + Cfg::oA);  // M diag(beta), strictly lower
  float* s_vec = reinterpret_cast<float*>(dsm + Cfg::oVec);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t bh = blockIdx.x / p.chunks, chunk = blockIdx.x - bh * p.chunks;
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int64_t t0 = chunk * kChunk;
  const int rows = (int)min((int64_t)kChunk, p.L - t0);

  pdl_wait();
  pdl_launch_dependents();
  const int64_t tok_stride = (int64_t)p.key_heads * p.dk;
  const int64_t first = (b * p.L + t0) * tok_stride + (int64_t)hk * p.dk;
  split_tile<T, NP, DKP>(s_k, static_cast<const T*>(p.k) + first, tok_stride, rows, p.dk / 8, tid);
  split_tile<T, NP, DKP>(s_q, static_cast<const T*>(p.q) + first, tok_stride, rows, p.dk / 8, tid);
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
    const int64_t tile = ((b * p.key_heads + hk) * p.chunks + chunk) * NP * (kChunk * DKP);
    bulk_s2g(p.k_tiles + tile, s_k, NP * TILE);
    bulk_s2g(p.q_tiles + tile, s_q, NP * TILE);
    bulk_commit();
  }

  // K K^T, then Q K^T, 16 rows a warp; tiles above the diagonal are not needed
  const int g4 = lane >> 2, t4 = lane & 3;
  const float* hi = s_vec + kVecCumHi * kChunk;
  const float* lo = s_vec + kVecCumLo * kChunk;
  const float* be = s_vec + kVecBeta * kChunk;
  auto with_k = [&](uint32_t rows_at, float (&acc)[8][4]) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[n][c] = 0.f;
#pragma unroll 2
    for (int kk = 0; kk < DKP / 16; ++kk) {
      uint32_t af[NP][4];
#pragma unroll
      for (int i = 0; i < NP; ++i) ldsm4(af[i], at_a<ROWB>(rows_at + i * TILE, lane, warp * 16, kk));
#pragma unroll
      for (int np2 = 0; np2 < 4; ++np2) {
        if (np2 > warp) break;
        Step<LV == 2, 2> s;
#pragma unroll
        for (int j = NP - 1; j >= 0; --j) {
          uint32_t bf[4];
          ldsm4(bf, at_b<ROWB>(s_k + j * TILE, lane, np2 * 16, kk));
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
  with_k(s_k, acc);
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = warp * 16 + g4 + r * 8, j0 = n * 8 + 2 * t4;
      float a[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j = j0 + c;
        a[c] = i > j ? acc[n][2 * r + c] * expf((hi[i] - hi[j]) + (lo[i] - lo[j])) * be[j] : 0.f;
      }
      *reinterpret_cast<float2*>(&s_a[i * kPad + j0]) = make_float2(a[0], a[1]);
    }
  with_k(s_q, acc);
  if (keeper) bulk_wait_read<0>();
  __syncthreads();  // K and Q are used up
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    uint32_t w[4][NS];  // P's 16 x 16 tile, in the order of an A operand
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = 2 * kk + (q >> 1), r = q & 1;
      const int i = warp * 16 + g4 + r * 8, j0 = n * 8 + 2 * t4;
      float v[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j = j0 + c;
        const float d = i == j ? 1.f : i > j ? expf((hi[i] - hi[j]) + (lo[i] - lo[j])) : 0.f;
        v[c] = i >= j ? acc[n][2 * r + c] * d * p.scale * be[j] : 0.f;
      }
      split_pair<NS>(v[0], v[1], w[q]);
    }
#pragma unroll
    for (int q = 0; q < NS; ++q) {
      const uint32_t a[4] = {w[0][q], w[1][q], w[2][q], w[3][q]};
      stsm4(at_a<MROW>(s_k + q * kMatBytes, lane, warp * 16, kk), a);
    }
  }
  fence_async();

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
  if (tid == 0) {  // every warp has written its rows of P
    bulk_s2g(p.p_mat + (bh * p.chunks + chunk) * NS * (kChunk * kChunk), s_k, NS * kMatBytes);
    bulk_commit();
  }
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

  const int64_t mat = (bh * p.chunks + chunk) * NS * (kChunk * kChunk);
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
      *reinterpret_cast<uint4*>(reinterpret_cast<char*>(p.n_mat + mat) +
                                tile_at<MROW>(q * kMatBytes, i, j0 / 8)) =
          make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
  }
  if (tid == 0) bulk_wait_all();
}

// ------------------------------------------------------------------ along the chunks
struct ScanParams {
  const __nv_bfloat16* q_tiles;
  const __nv_bfloat16* k_tiles;
  const void* v;
  const __nv_bfloat16* n_mat;
  const __nv_bfloat16* p_mat;
  const float* vecs;
  const float* initial;
  float* final_state;
  void* out;                  // KEEP false
  __nv_bfloat16* e_parts;     // KEEP true: strips [head][chunk][dv / 16][NS], as in shared memory
  __nv_bfloat16* s_parts;     // [head][chunk][dv / 16][half of dk][NS][16][DKP / 2]
  int64_t L, chunks;
  int key_heads, heads, dk, dv, slices;
  float scale;
};

// KEEP: no output; E and the states entering the chunks are written as parts
// (what the backward pass multiplies with).
template <typename T, int NP, int LV, int DKP, int NW, bool KEEP>
struct ScanCfg {
  static constexpr int NS = LV + 1;
  // parts of S0 and E that leave the chain warps: outputs of 16 bits need two
  static constexpr int NO = KEEP ? NS : sizeof(T) == 4 ? 3 : 2;
  static constexpr int kThreads = (KEEP ? 2 * NW + 1 : 3 * NW) * 32;
  static constexpr int kTileK = kChunk * DKP * 2;
  static constexpr int oN = NP * kTileK, oVec = oN + NS * kMatBytes;
  static constexpr int kStageK = oVec + 3 * kChunk * 4;  // enter, leave, beta
  static constexpr int oP = NP * kTileK, oEnter = oP + NO * kMatBytes;
  static constexpr int kStageQ = KEEP ? 0 : oEnter + 256;
  static constexpr int kV = kChunk * 16 * (int)sizeof(T);
  // of a strip: v twice; S0's parts; two halves of K S0^T, later E; E's parts or O
  static constexpr int kXS = NO * 16 * DKP * 2, kHalf = 8 * 512;
  static constexpr int kXE = KEEP ? NS * kStrip : sizeof(T) == 2 ? kStrip : 0;  // else: O's
  static constexpr int kWarp = 2 * kV + kXS + 2 * kHalf + kXE;
  static constexpr int kRoom = 227 * 1024 - 1280;        // barriers, alignment
  static constexpr int kStK = NW * kWarp + 2 * kStageK + kStageQ <= kRoom ? 2 : 1;
  static constexpr int kStQ = KEEP ? 1 : NW * kWarp + kStK * kStageK + 2 * kStageQ <= kRoom ? 2 : 1;
  static constexpr int oQ = kStK * kStageK, oWarp = oQ + kStQ * kStageQ;
  static constexpr int kSmem = oWarp + NW * kWarp + 128;
  static_assert(kStageK % 128 == 0 && kStageQ % 128 == 0 && kSmem + 1152 <= 227 * 1024);
};

template <typename T, int NP, int LV, int DKP, int NW, bool KEEP>
__global__ void __launch_bounds__(ScanCfg<T, NP, LV, DKP, NW, KEEP>::kThreads, 1)
    delta_scan_kernel(const ScanParams p) {
  using Cfg = ScanCfg<T, NP, LV, DKP, NW, KEEP>;
  constexpr int NS = Cfg::NS, NO = Cfg::NO, LO = NO - 1, ROWB = DKP * 2, NT = DKP / 8;
  constexpr int MROW = kChunk * 2;  // bytes of a row of N and P
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t sm0 = smem_addr(dsm);
  // full: the copies of a stage have landed / the chain warp has written;
  // free: whoever reads a stage or a buffer is done with it
  __shared__ __align__(8) uint64_t full_k[2], free_k[2], full_q[2], free_q[2];
  __shared__ __align__(8) uint64_t full_s[NW], free_s[NW], full_e[NW], free_e[NW], pair[NW];
  __shared__ int s_bad[NW];
  __shared__ int s_spoilt[NW][16];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int64_t bh = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - bh * p.slices);
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int dv_cta = slice * NW * 16;
  const int nact = min(NW, (p.dv - dv_cta + 15) / 16);  // strips with values
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&full_k[i], 1);
      mbar_init(&free_k[i], 2 * nact);
      mbar_init(&full_q[i], 1);
      mbar_init(&free_q[i], nact);
    }
    for (int i = 0; i < NW; ++i) {
      mbar_init(&full_s[i], 2);
      mbar_init(&free_s[i], 1);
      mbar_init(&full_e[i], 2);
      mbar_init(&free_e[i], 1);
      mbar_init(&pair[i], 2);
    }
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();

  const int64_t unit0 = bh * p.chunks;
  // loads of a chunk's stages; `free` waits until the stage's last reader is done
  const int64_t tile = (b * p.key_heads + hk) * p.chunks;
  int64_t next_k = 0, next_q = 0;  // chunks issued (by the one lane that loads)
  auto issue_k = [&]() {
    const int64_t c = next_k;
    const int s = (int)(c % Cfg::kStK);
    if (c >= Cfg::kStK && !mbar_wait_bounded(&free_k[s], (uint32_t)((c / Cfg::kStK - 1) & 1)))
      return false;
    const uint32_t st = sm0 + s * Cfg::kStageK;
    mbar_expect_tx(&full_k[s], Cfg::oVec + 3 * kChunk * 4);
    bulk_in(st, p.k_tiles + (tile + c) * NP * (kChunk * DKP), NP * Cfg::kTileK, &full_k[s]);
    bulk_in(st + Cfg::oN, p.n_mat + (unit0 + c) * NS * (kChunk * kChunk), NS * kMatBytes, &full_k[s]);
    bulk_in(st + Cfg::oVec, p.vecs + (unit0 + c) * (kVecCount * kChunk), 3 * kChunk * 4, &full_k[s]);
    ++next_k;
    return true;
  };
  auto issue_q = [&]() {
    const int64_t c = next_q;
    const int s = (int)(c % Cfg::kStQ);
    if (c >= Cfg::kStQ && !mbar_wait_bounded(&free_q[s], (uint32_t)((c / Cfg::kStQ - 1) & 1)))
      return false;
    const uint32_t st = sm0 + Cfg::oQ + s * Cfg::kStageQ;
    mbar_expect_tx(&full_q[s], Cfg::oEnter + kChunk * 4);
    bulk_in(st, p.q_tiles + (tile + c) * NP * (kChunk * DKP), NP * Cfg::kTileK, &full_q[s]);
    bulk_in(st + Cfg::oP, p.p_mat + (unit0 + c) * NS * (kChunk * kChunk), NO * kMatBytes, &full_q[s]);
    bulk_in(st + Cfg::oEnter, p.vecs + (unit0 + c) * (kVecCount * kChunk), kChunk * 4, &full_q[s]);
    ++next_q;
    return true;
  };
  // After a wait that gave up: no copy may land after the CTA is gone.
  auto drain = [&]() {
    for (int64_t j = max((int64_t)0, next_k - Cfg::kStK); j < next_k; ++j)
      mbar_wait_bounded(&full_k[j % Cfg::kStK], (uint32_t)((j / Cfg::kStK) & 1));
    for (int64_t j = max((int64_t)0, next_q - Cfg::kStQ); j < next_q; ++j)
      mbar_wait_bounded(&full_q[j % Cfg::kStQ], (uint32_t)((j / Cfg::kStQ) & 1));
  };
  if (KEEP && warp == 2 * NW) {
    // ---------------------------------------------------------- loader
    if (lane == 0) {
      bool ok = true;
      while (ok && next_k < p.chunks) ok = issue_k();
      if (!ok) drain();
    }
  } else if (warp < 2 * NW) {
    // ---------------------------------------------------------- chain
    const int w = warp >> 1, side = warp & 1;  // strip, half of dk
    const int dv0 = dv_cta + w * 16;
    const int nval = p.dv - dv0;  // values of the strip's 16 rows that exist (may be <= 0)
    if (nval > 0) {
      constexpr int HT = NT / 2;  // tiles of this half
      const int d0 = side * (DKP / 2);
      const int64_t vstride = (int64_t)p.heads * p.dv;
      const uint32_t own = sm0 + Cfg::oWarp + w * Cfg::kWarp;
      const uint32_t x_s = own + 2 * Cfg::kV, x_h = x_s + Cfg::kXS, x_e = x_h + 2 * Cfg::kHalf;
      // E's tiles: blocks of 16 tokens 0, 3 are side 0's, 1, 2 side 1's (five
      // products of 16 x 16 blocks each).  A side leaves them where the other's
      // half of K S0^T was, which only it has read; of the two sides only the
      // other reads them (and writes there next).
      auto e_at = [&](int n) {
        const int blk = n >> 1, of = blk == 0 || blk == 3 ? 0 : 1;
        return x_h + (1 - of) * Cfg::kHalf + ((blk >> 1) * 2 + (n & 1)) * 512 + lane * 16;
      };
      const char* v_next = reinterpret_cast<const char*>(static_cast<const T*>(p.v) +
                                                         b * p.L * vstride + (int64_t)h * p.dv + dv0);
      const int vunits = min(16, nval) * (int)sizeof(T) / 16;
      const bool loads = warp == 0 && lane == 0;
      if (!KEEP && loads)
        while (next_k < min((int64_t)Cfg::kStK, p.chunks)) issue_k();
      __syncwarp();
      auto load_v = [&](int64_t c) {  // side s loads rows 32 s..
        constexpr int U = (int)sizeof(T);
        const int rows = (int)min((int64_t)kChunk, p.L - c * kChunk);
        const uint32_t dst = own + (int)(c & 1) * Cfg::kV;
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int r = side * 32 + (i * 32 + lane) / U, u = (i * 32 + lane) % U;
          const bool in = r < rows && u < vunits;
          cp16(U == 2 ? strip_at(dst, r, u) : strip32_at(dst, r, u),
               in ? v_next + r * (vstride * (int)sizeof(T)) + u * 16 : v_next, in);
        }
        v_next += kChunk * vstride * (int)sizeof(T);
        cp_commit();
      };
      load_v(0);

      float S[HT][4];
#pragma unroll
      for (int n = 0; n < HT; ++n) {
#pragma unroll
        for (int c = 0; c < 4; ++c) S[n][c] = 0.f;
        if (p.initial != nullptr) {
          const int dk = d0 + n * 8 + 2 * t4;
          const float* src = p.initial + (bh * p.dv + dv0 + g4) * p.dk + dk;
          if (dk < p.dk) {
            const float2 v = *reinterpret_cast<const float2*>(src);
            S[n][0] = v.x;
            S[n][1] = v.y;
            if (nval > 8) {
              const float2 y = *reinterpret_cast<const float2*>(src + 8 * p.dk);
              S[n][2] = y.x;
              S[n][3] = y.y;
            }
          }
        }
      }

      bool ok = true;
      for (int64_t c = 0; c < p.chunks; ++c) {
        const int sk = (int)(c % Cfg::kStK);
        const uint32_t st = sm0 + sk * Cfg::kStageK;
        const float* vec = reinterpret_cast<const float*>(dsm + sk * Cfg::kStageK + Cfg::oVec);
        const float* enter = vec + kVecEnter * kChunk;
        const float* leave = vec + kVecLeave * kChunk;
        const float* beta = vec + kVecBeta * kChunk;
        // one stage: the load waits for every chain warp
        if (!KEEP && Cfg::kStK == 1 && c > 0 && loads) ok = issue_k();
        ok = ok && mbar_wait_bounded(&full_k[sk], (uint32_t)((c / Cfg::kStK) & 1));
        if (!KEEP && c > 0) {
          ok = ok && mbar_wait_bounded(&free_s[w], (uint32_t)((c - 1) & 1));
          ok = ok && mbar_wait_bounded(&free_e[w], (uint32_t)((c - 1) & 1));
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const float total = enter[kChunk - 1];
        if (KEEP) {  // S0's parts of the chunk before have been read
          if (lane == 0) bulk_wait_read<1>();
          __syncwarp();
        }

        // X = (K S0^T)^T: 16 values x 64 tokens, this half of dk.  S0's parts
        // go to shared memory.
        float X[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) X[n][e] = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < HT / 2; ++k2) {
          const int kk = side * (HT / 2) + k2;
          uint32_t a[NS][4];
          split_frag<NS>(S[2 * k2], S[2 * k2 + 1], a);
#pragma unroll
          for (int q = 0; q < NO; ++q)
            stsm4(half_a<DKP>(x_s + (side * NO + q) * 16 * DKP, lane, k2), a[q]);
#pragma unroll
          for (int n2 = 0; n2 < 4; ++n2) {
            Step<LV == 2, 2> s;
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) {
              uint32_t kb[4];
              ldsm4(kb, at_b<ROWB>(st + i * Cfg::kTileK, lane, n2 * 16, kk));
#pragma unroll
              for (int j = LV - i; j >= 0; --j) {
                s.mma(0, X[2 * n2], a[j], kb[0], kb[1]);
                s.mma(1, X[2 * n2 + 1], a[j], kb[2], kb[3]);
              }
            }
            s.add(0, X[2 * n2]);
            s.add(1, X[2 * n2 + 1]);
          }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) sts_acc(x_h + side * Cfg::kHalf + n * 512 + lane * 16, X[n]);
        if (KEEP) fence_async();
        cp_wait<0>();  // this side's rows of v
        __syncwarp();
        if (KEEP && lane == 0) {
          bulk_s2g(p.s_parts + (((unit0 + c) * ((p.dv + 15) / 16) + dv0 / 16) * 2 + side) * NS * 8 * DKP,
                   x_s + side * NS * 16 * DKP, NS * 16 * DKP);
          bulk_commit();
        }
        if (lane == 0) {
          mbar_arrive(&pair[w]);
          if (!KEEP) mbar_arrive(&full_s[w]);
        }
        // the stage of the chunk before is free by now, or nearly
        if (!KEEP && Cfg::kStK == 2 && loads && c > 0 && next_k < p.chunks) ok = issue_k();
        ok = ok && mbar_wait_bounded(&pair[w], 0);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;

        // R = V - exp(G) X, in place; both sides add the halves in the same order
        const uint32_t vst = own + (int)(c & 1) * Cfg::kV;
#pragma unroll
        for (int n2 = 0; n2 < 4; ++n2) {
          uint32_t vb[4];
          if constexpr (sizeof(T) == 2) ldsm4_t(vb, strip_at_t(vst, lane, n2));
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int n = 2 * n2 + half, tok = n * 8 + 2 * t4;
            const float2 ge = *reinterpret_cast<const float2*>(enter + tok);
            float v[4], y[4];
            lds_acc(x_h + (1 - side) * Cfg::kHalf + n * 512 + lane * 16, y);
            if constexpr (sizeof(T) == 2) {
              const float2 lo = unpack2<T>(vb[2 * half]), hi = unpack2<T>(vb[2 * half + 1]);
              v[0] = lo.x;
              v[1] = lo.y;
              v[2] = hi.x;
              v[3] = hi.y;
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int col = g4 + (e >> 1) * 8;
                const uint32_t at = strip32_at(vst, tok + (e & 1), col / 4) + (col % 4) * 4;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[e]) : "r"(at) : "memory");
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) X[n][e] = fmaf(-((e & 1) ? ge.y : ge.x), X[n][e] + y[e], v[e]);
          }
        }
        if (c + 1 < p.chunks) load_v(c + 1);  // the buffer of the chunk before

        // An infinity or a NaN in R (of v, k, or the state) spoils its row of
        // values from that token on, but the zeros above the diagonals of N
        // and P would carry it to earlier tokens: it is taken out here and
        // put back into E, O and the state afterwards.
        int spoilt[2] = {kChunk, kChunk};  // first such token of the thread's two rows
        float probe[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) probe[e] = fmaf(X[n][e], 0.f, probe[e]);
        const bool bad =
            __any_sync(0xffffffffu, (probe[0] + probe[1]) + (probe[2] + probe[3]) != 0.f);
        if (bad) {
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(fabsf(X[n][e]) <= 3.4e38f))
                spoilt[e >> 1] = min(spoilt[e >> 1], n * 8 + 2 * t4 + (e & 1));
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            spoilt[r] = min(spoilt[r], __shfl_xor_sync(0xffffffffu, spoilt[r], 1));
            spoilt[r] = min(spoilt[r], __shfl_xor_sync(0xffffffffu, spoilt[r], 2));
          }
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n * 8 + 2 * t4 + (e & 1) >= spoilt[e >> 1]) X[n][e] = 0.f;
        }

        // E = N R, this side's blocks of tokens: 0, 3 or 1, 2
        float E[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) E[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t a[NS][4];
          split_frag<NS>(X[2 * kk], X[2 * kk + 1], a);
          auto block = [&](int n2, float (&e0)[4], float (&e1)[4]) {
            Step<LV == 2, 2> s;
#pragma unroll
            for (int i = LV; i >= 0; --i) {
              uint32_t nb[4];
              ldsm4(nb, at_b<MROW>(st + Cfg::oN + i * kMatBytes, lane, n2 * 16, kk));
#pragma unroll
              for (int j = LV - i; j >= 0; --j) {
                s.mma(0, e0, a[j], nb[0], nb[1]);
                s.mma(1, e1, a[j], nb[2], nb[3]);
              }
            }
            s.add(0, e0);
            s.add(1, e1);
          };
          if (kk <= side) block(side, E[0], E[1]);
          if (kk <= 3 - side) block(3 - side, E[2], E[3]);
        }
        // E's tiles go to the other side and the output warp
        if (KEEP) {  // E's parts of the chunk before have been read
          if (lane == 0) bulk_wait_read<1>();
          __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n2 = i == 0 ? side : 3 - side;
          sts_acc(e_at(2 * n2), E[2 * i]);
          sts_acc(e_at(2 * n2 + 1), E[2 * i + 1]);
          if (KEEP) {
            if (bad) {
#pragma unroll
              for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (n2 * 16 + n * 8 + 2 * t4 + (e & 1) >= spoilt[e >> 1])
                    E[2 * i + n][e] = __int_as_float(0x7fc00000);
            }
            uint32_t a[NS][4];
            split_frag<NS>(E[2 * i], E[2 * i + 1], a);
#pragma unroll
            for (int q = 0; q < NS; ++q) stsm4_t(strip_at_t(x_e + q * kStrip, lane, n2), a[q]);
          }
        }
        if (KEEP) {
          fence_async();
          __syncwarp();
          if (lane == 0) {
            __nv_bfloat16* ep =
                p.e_parts + ((unit0 + c) * ((p.dv + 15) / 16) + dv0 / 16) * NS * (kStrip / 2);
#pragma unroll
            for (int q = 0; q < NS; ++q)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int n2 = i == 0 ? side : 3 - side;  // 16 rows of 32 bytes
                bulk_s2g(ep + q * (kStrip / 2) + n2 * 256, x_e + q * kStrip + n2 * 512, 512);
              }
            bulk_commit();
          }
        } else {
          if (side == 0 && lane == 0) s_bad[w] = bad;
          if (side == 0 && bad && t4 == 0) {
            s_spoilt[w][g4] = spoilt[0];
            s_spoilt[w][g4 + 8] = spoilt[1];
          }
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&pair[w]);
          if (!KEEP) mbar_arrive(&full_e[w]);
        }
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&pair[w], 1));
        if (!ok) break;

        // S = exp(G_C) S + (beta exp(G_C - G) E)^T K, this half of dk.  The
        // chunk's sum starts at zero and joins the state in one rounded
        // multiply-add.
        uint32_t u[4][NS][4];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          float f[2][4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int n = 2 * kk + half, tok = n * 8 + 2 * t4;
            const float2 lv = *reinterpret_cast<const float2*>(leave + tok);
            const float2 bt = *reinterpret_cast<const float2*>(beta + tok);
            const float w0 = lv.x * bt.x, w1 = lv.y * bt.y;
            if ((kk == side) | (kk == 3 - side)) {
#pragma unroll
              for (int e = 0; e < 4; ++e) f[half][e] = E[(kk >> 1) * 2 + half][e];
            } else {
              lds_acc(e_at(n), f[half]);
            }
            f[half][0] *= w0;
            f[half][1] *= w1;
            f[half][2] *= w0;
            f[half][3] *= w1;
          }
          split_frag<NS>(f[0], f[1], u[kk]);
        }
#pragma unroll
        for (int n4 = 0; n4 < HT / 4; ++n4) {
          float d[4][4];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            Step<LV == 2, 4> s;
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) {
              uint32_t b0[4], b1[4];
              ldsm4_t(b0, at_bt<ROWB>(st + i * Cfg::kTileK, lane, d0 + n4 * 32, kk));
              ldsm4_t(b1, at_bt<ROWB>(st + i * Cfg::kTileK, lane, d0 + n4 * 32 + 16, kk));
#pragma unroll
              for (int j = LV - i; j >= 0; --j) {
                s.mma(0, d[0], u[kk][j], b0[0], b0[1]);
                s.mma(1, d[1], u[kk][j], b0[2], b0[3]);
                s.mma(2, d[2], u[kk][j], b1[0], b1[1]);
                s.mma(3, d[3], u[kk][j], b1[2], b1[3]);
              }
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) s.add(n, d[n]);
          }
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[n4 * 4 + n][e] = fmaf(total, S[n4 * 4 + n][e], d[n][e]);
        }
        if (bad)
#pragma unroll
          for (int n = 0; n < HT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (spoilt[e >> 1] < kChunk) S[n][e] = __int_as_float(0x7fc00000);
        warp_arrive(&free_k[sk], lane);
      }

      cp_wait<0>();
      if (!ok && loads) drain();
      if (KEEP) {
        if (lane == 0) bulk_wait_all();
      } else if (ok && p.final_state != nullptr) {
#pragma unroll
        for (int n = 0; n < HT; ++n) {
          const int dk = d0 + n * 8 + 2 * t4;
          float* dst = p.final_state + (bh * p.dv + dv0 + g4) * p.dk + dk;
          if (dk < p.dk) {
            *reinterpret_cast<float2*>(dst) = make_float2(S[n][0], S[n][1]);
            if (nval > 8) *reinterpret_cast<float2*>(dst + 8 * p.dk) = make_float2(S[n][2], S[n][3]);
          }
        }
      }
    }
  } else if (!KEEP) {
    // ---------------------------------------------------------- output
    const int w = warp - 2 * NW;
    const int dv0 = dv_cta + w * 16;
    const int nval = p.dv - dv0;
    if (nval > 0) {
      const int64_t vstride = (int64_t)p.heads * p.dv;
      const uint32_t x_s = sm0 + Cfg::oWarp + w * Cfg::kWarp + 2 * Cfg::kV, x_h = x_s + Cfg::kXS,
                     x_o = x_h + 2 * Cfg::kHalf;
      const bool loads = w == 0 && lane == 0;
      if (loads) {
        while (next_q < min((int64_t)Cfg::kStQ, p.chunks)) issue_q();
      }
      __syncwarp();
      bool ok = true;
      for (int64_t c = 0; c < p.chunks; ++c) {
        const int sq = (int)(c % Cfg::kStQ);
        const uint32_t st = sm0 + Cfg::oQ + sq * Cfg::kStageQ;
        const float* enter = reinterpret_cast<const float*>(dsm + Cfg::oQ + sq * Cfg::kStageQ + Cfg::oEnter);
        ok = mbar_wait_bounded(&full_q[sq], (uint32_t)((c / Cfg::kStQ) & 1));
        ok = ok && mbar_wait_bounded(&full_s[w], (uint32_t)(c & 1));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        float O[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) O[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DKP / 16; ++kk) {
          uint32_t a[NO][4];
#pragma unroll
          for (int q = 0; q < NO; ++q)
            ldsm4(a[q], half_a<DKP>(x_s + (kk / (DKP / 32) * NO + q) * 16 * DKP, lane, kk % (DKP / 32)));
#pragma unroll
          for (int n2 = 0; n2 < 4; ++n2) {
            Step<LO == 2, 2> s;
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) {
              if (i > LO) continue;
              uint32_t qb[4];
              ldsm4(qb, at_b<ROWB>(st + i * Cfg::kTileK, lane, n2 * 16, kk));
#pragma unroll
              for (int j = LO - i; j >= 0; --j) {
                s.mma(0, O[2 * n2], a[j], qb[0], qb[1]);
                s.mma(1, O[2 * n2 + 1], a[j], qb[2], qb[3]);
              }
            }
            s.add(0, O[2 * n2]);
            s.add(1, O[2 * n2 + 1]);
          }
        }
        warp_arrive(&free_s[w], lane);
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          const float2 ge = *reinterpret_cast<const float2*>(enter + n * 8 + 2 * t4);
          O[n][0] *= ge.x * p.scale;
          O[n][1] *= ge.y * p.scale;
          O[n][2] *= ge.x * p.scale;
          O[n][3] *= ge.y * p.scale;
        }
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full_e[w], (uint32_t)(c & 1)));
        if (!ok) break;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          float e0[4], e1[4];  // where the chain's e_at puts them
          const uint32_t e_blk = x_h + (kk == 0 || kk == 3 ? Cfg::kHalf : 0) + (kk >> 1) * 1024 + lane * 16;
          lds_acc(e_blk, e0);
          lds_acc(e_blk + 512, e1);
          uint32_t a[NO][4];
          split_frag<NO>(e0, e1, a);
#pragma unroll
          for (int n2 = kk; n2 < 4; ++n2) {
            Step<LO == 2, 2> s;
#pragma unroll
            for (int i = LO; i >= 0; --i) {
              uint32_t pb[4];
              ldsm4(pb, at_b<MROW>(st + Cfg::oP + i * kMatBytes, lane, n2 * 16, kk));
#pragma unroll
              for (int j = LO - i; j >= 0; --j) {
                s.mma(0, O[2 * n2], a[j], pb[0], pb[1]);
                s.mma(1, O[2 * n2 + 1], a[j], pb[2], pb[3]);
              }
            }
            s.add(0, O[2 * n2]);
            s.add(1, O[2 * n2 + 1]);
          }
        }
        const bool bad = s_bad[w] != 0;
        const int first[2] = {s_spoilt[w][g4], s_spoilt[w][g4 + 8]};
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&free_q[sq]);
          mbar_arrive(&free_e[w]);
        }
        if (bad) {
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n * 8 + 2 * t4 + (e & 1) >= first[e >> 1]) O[n][e] = __int_as_float(0x7fc00000);
        }
        const int64_t t0 = c * kChunk;
        T* out = static_cast<T*>(p.out) + (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv0;
        const int rows = (int)min((int64_t)kChunk, p.L - t0);
        if constexpr (sizeof(T) == 2) {
          // through shared memory, transposed, for stores of 16 bytes
          __syncwarp();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t a[4] = {pack2<T>(O[2 * kk][0], O[2 * kk][1]), pack2<T>(O[2 * kk][2], O[2 * kk][3]),
                                   pack2<T>(O[2 * kk + 1][0], O[2 * kk + 1][1]),
                                   pack2<T>(O[2 * kk + 1][2], O[2 * kk + 1][3])};
            stsm4_t(strip_at_t(x_o, lane, kk), a);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i * 16 + (lane >> 1), un = lane & 1;
            if (r < rows && un * 8 < nval)
              *reinterpret_cast<uint4*>(out + r * vstride + un * 8) = lds128(strip_at(x_o, r, un));
          }
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n)
            store_t<T>(out + (int64_t)n * 8 * vstride, vstride, O[n], lane, rows - n * 8, nval);
        }
        if (loads && next_q < p.chunks) ok = issue_q();
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (loads && !ok) drain();
    }
  }
  __syncthreads();  // shared memory outlives every copy into it
}

// ------------------------------------------------------------------ host side
template <typename Kern>
cudaError_t configure(Kern kern, int smem) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
}

template <typename T, int LV, int DKP, int NW, bool KEEP>
cudaError_t scan_nw(const DeltaArgs& a, ScanParams& p, int64_t bh) {
  using Cfg = ScanCfg<T, kParts<T>, LV, DKP, NW, KEEP>;
  auto kern = delta_scan_kernel<T, kParts<T>, LV, DKP, NW, KEEP>;
  const cudaError_t e = configure(kern, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  p.slices = (int)((a.dv + NW * 16 - 1) / (NW * 16));
  return launch_pdl(kern, (unsigned)(bh * p.slices), Cfg::kThreads, Cfg::kSmem, a.stream, p);
}

}  // namespace

// Prep and scan for sequences [b0, b0 + nb) of the call.  keep: for the
// backward pass (E and the states instead of the output).
template <typename T, int LV, int DKP>
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
  pp.q_tiles = bf(pl.q_tiles);
  pp.k_tiles = bf(pl.k_tiles);
  pp.log_decay = static_cast<const T*>(a.log_decay) + g0;
  pp.beta = static_cast<const T*>(a.beta) + g0;
  pp.n_mat = bf(pl.n_mat);
  pp.p_mat = bf(pl.p_mat);
  pp.vecs = reinterpret_cast<float*>(ws + pl.vecs);
  pp.L = a.seqlen;
  pp.chunks = pl.chunks;
  pp.key_heads = (int)a.key_heads;
  pp.heads = (int)a.heads;
  pp.dk = (int)a.dk;
  pp.scale = a.scale;
  auto prep = delta_prep_kernel<T, NP, LV, DKP>;
  constexpr int prep_smem = PrepCfg<NP, LV + 1, DKP>::kSmem;
  cudaError_t e = configure(prep, prep_smem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(prep, (unsigned)(bh * pl.chunks), kPrepThreads, prep_smem, a.stream, pp);
  if (e != cudaSuccess) return e;

  ScanParams p{};
  p.q_tiles = pp.q_tiles;
  p.k_tiles = pp.k_tiles;
  p.v = static_cast<const T*>(a.v) + v0;
  p.n_mat = pp.n_mat;
  p.p_mat = pp.p_mat;
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
  // Strips per CTA: 4, or 2 where that still leaves an SM to every CTA
  // (and for fp32, whose tiles leave room for no more).
  const bool two = sizeof(T) == 4 || bh * ((a.dv + 31) / 32) <= a.num_sms;
  if constexpr (sizeof(T) == 4) {
    return keep ? scan_nw<T, LV, DKP, 2, true>(a, p, bh) : scan_nw<T, LV, DKP, 2, false>(a, p, bh);
  } else {
    if (keep)
      return two ? scan_nw<T, LV, DKP, 2, true>(a, p, bh) : scan_nw<T, LV, DKP, 4, true>(a, p, bh);
    return two ? scan_nw<T, LV, DKP, 2, false>(a, p, bh) : scan_nw<T, LV, DKP, 4, false>(a, p, bh);
  }
}

template cudaError_t delta_fwd_pass<__nv_bfloat16, 1, 64>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__nv_bfloat16, 1, 128>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__nv_bfloat16, 2, 64>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__nv_bfloat16, 2, 128>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__half, 1, 64>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__half, 1, 128>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__half, 2, 64>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<__half, 2, 128>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<float, 2, 64>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);
template cudaError_t delta_fwd_pass<float, 2, 128>(const DeltaArgs&, const DeltaPlan&, int64_t, int64_t, bool);

DeltaPlan delta_plan(int64_t batch, int64_t seqlen, int64_t key_heads, int64_t heads, int64_t dk,
                     int64_t dv, int dtype, bool wide, bool backward) {
  DeltaPlan pl{};
  pl.np = dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1;
  pl.ns = wide || dtype == kF32 ? 3 : 2;
  pl.dkp = dk <= 64 ? 64 : 128;
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
    const int64_t tiles = nb * key_heads * pl.chunks * pl.np * kChunk * pl.dkp * 2;
    pl.q_tiles = take(tiles);
    pl.k_tiles = take(tiles);
    pl.n_mat = take(c * pl.ns * kChunk * kChunk * 2);
    pl.p_mat = take(c * pl.ns * kChunk * kChunk * 2);
    pl.vecs = take(c * kVecCount * kChunk * 4);
    if (backward) {
      const int64_t strips = (dv + 15) / 16;
      if (pl.np > 1) pl.grad_rows = take(pl.np * tok * heads * dv * 2);
      pl.do_parts = take(c * pl.np * kStrip * strips);
      pl.e_parts = take(c * pl.ns * kStrip * strips);
      pl.dv_parts = take(c * pl.ns * kStrip * strips);
      pl.s_parts = take(c * pl.ns * strips * 16 * pl.dkp * 2);
      pl.ds_parts = take(c * pl.ns * strips * 16 * pl.dkp * 2);
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
    const cudaError_t e = pl.dkp == 64 ? delta_fwd_pass<T, LV, 64>(a, pl, b0, nb, false)
                                       : delta_fwd_pass<T, LV, 128>(a, pl, b0, nb, false);
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
