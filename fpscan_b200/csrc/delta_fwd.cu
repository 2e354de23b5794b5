// Gated delta rule, forward over a sequence in chunks of 64 tokens (sm_100a).
// The mathematics and the number format of the products are in delta.cuh.
//
//   delta_split_kernel  fp16 / fp32 inputs only: cuts q, k into bf16 parts.
//   delta_prep_kernel   one CTA per (chunk, head), all in parallel: the
//                       64 x 64 matrices N and P and the decay vectors.
//   delta_scan_kernel   runs along the chunks of a head with the state in
//                       registers: the only sequential part.
//
// The scan keeps the state transposed, S^T tiles as accumulators: a warp
// owns 16 rows of values (dv) and all of dk (64 registers a thread at
// dk = 128).  Every product of the chain then has the warp's own rows as its
// A operand -- K S0^T, N R, P E, the state's update -- and an accumulator
// turns into the next product's A operand by packing registers, so the
// chain of a chunk runs without shared memory or a barrier between its
// products; K, Q, N and P are the B operands and come from shared memory
// once for all warps.  Columns of the state never mix, so a head may be cut
// along dv over as many CTAs as the GPU has room for.
#include <algorithm>

#include "delta.cuh"
#include "internal.h"

namespace fpscan {

namespace {

// ------------------------------------------------------------------ input parts
struct SplitParams {
  const void* src[3];
  __nv_bfloat16* dst[3];
  int64_t n[3];       // elements (multiples of 8)
};

template <typename T>
__global__ void __launch_bounds__(256) delta_split_kernel(const SplitParams p) {
  constexpr int NP = kParts<T>;
  pdl_wait();
  pdl_launch_dependents();
  const int which = blockIdx.x % 3;
  const int64_t n = p.n[which], step = (int64_t)(gridDim.x / 3) * blockDim.x * 8;
  const T* src = static_cast<const T*>(p.src[which]);
  __nv_bfloat16* dst = p.dst[which];
  for (int64_t i = ((int64_t)(blockIdx.x / 3) * blockDim.x + threadIdx.x) * 8; i < n; i += step) {
    float x[8];
    constexpr int V = Elem<T>::kVec;
#pragma unroll
    for (int j = 0; j < 8 / V; ++j) {
      Vec16<T> v;
      v.raw = *reinterpret_cast<const uint4*>(src + i + j * V);
#pragma unroll
      for (int c = 0; c < V; ++c) x[j * V + c] = Elem<T>::load(v.e[c]);
    }
    uint32_t w[4][NP];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_pair<NP>(x[2 * j], x[2 * j + 1], w[j]);
#pragma unroll
    for (int q = 0; q < NP; ++q)
      *reinterpret_cast<uint4*>(dst + q * n + i) = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
  }
}

// ------------------------------------------------------------------ per-chunk matrices
struct PrepParams {
  const __nv_bfloat16* q;   // parts, part p at + p * part_stride
  const __nv_bfloat16* k;
  int64_t part_stride;
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
constexpr int kPad = kChunk + 1;  // fp32 rows in shared memory: columns on distinct banks

template <int NP, int DKP>
constexpr int prep_smem() {
  return 2 * NP * kChunk * DKP * 2 + 2 * kChunk * kPad * 4 + kVecCount * kChunk * 4 + 128;
}

template <typename T, int NP, int LV, int DKP>
__global__ void __launch_bounds__(kPrepThreads) delta_prep_kernel(const PrepParams p) {
  constexpr int NS = LV + 1;
  constexpr int ROWB = DKP * 2, TILE = kChunk * ROWB;
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t s_k = smem_addr(dsm), s_q = s_k + NP * TILE;
  float* s_a = reinterpret_cast<float*>(dsm + 2 * NP * TILE);  // M diag(beta), strictly lower
  float* s_n = s_a + kChunk * kPad;                            // its unit-triangle inverse
  float* s_vec = s_n + kChunk * kPad;

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
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    load_tile<kChunk, ROWB, kPrepThreads>(s_k + q * TILE, p.k + q * p.part_stride + first,
                                          tok_stride * 2, rows, p.dk / 8, tid);
    load_tile<kChunk, ROWB, kPrepThreads>(s_q + q * TILE, p.q + q * p.part_stride + first,
                                          tok_stride * 2, rows, p.dk / 8, tid);
  }
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
  __syncthreads();

  // K K^T and Q K^T, 16 rows a warp; tiles above the diagonal are not needed
  const int g4 = lane >> 2, t4 = lane & 3;
  float kk_acc[8][4], qk_acc[8][4];
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int c = 0; c < 4; ++c) kk_acc[n][c] = qk_acc[n][c] = 0.f;
#pragma unroll 2
  for (int kk = 0; kk < DKP / 16; ++kk) {
    uint32_t ka[NP][4], qa[NP][4];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      ldsm4(ka[i], at_a<ROWB>(s_k + i * TILE, lane, warp * 16, kk));
      ldsm4(qa[i], at_a<ROWB>(s_q + i * TILE, lane, warp * 16, kk));
    }
#pragma unroll
    for (int np2 = 0; np2 < 4; ++np2) {
      if (np2 > warp) break;
      Step<LV == 2, 4> s;
#pragma unroll
      for (int j = NP - 1; j >= 0; --j) {
        uint32_t bf[4];
        ldsm4(bf, at_b<ROWB>(s_k + j * TILE, lane, np2 * 16, kk));
#pragma unroll
        for (int i = NP - 1; i >= 0; --i) {
          if (i + j > LV) continue;
          s.mma(0, kk_acc[2 * np2], ka[i], bf[0], bf[1]);
          s.mma(1, kk_acc[2 * np2 + 1], ka[i], bf[2], bf[3]);
          s.mma(2, qk_acc[2 * np2], qa[i], bf[0], bf[1]);
          s.mma(3, qk_acc[2 * np2 + 1], qa[i], bf[2], bf[3]);
        }
      }
      s.add(0, kk_acc[2 * np2]);
      s.add(1, kk_acc[2 * np2 + 1]);
      s.add(2, qk_acc[2 * np2]);
      s.add(3, qk_acc[2 * np2 + 1]);
    }
  }
  const float* hi = s_vec + kVecCumHi * kChunk;
  const float* lo = s_vec + kVecCumLo * kChunk;
  const float* be = s_vec + kVecBeta * kChunk;
  const int64_t mat = (bh * p.chunks + chunk) * NS * (kChunk * kChunk);
#pragma unroll
  for (int n = 0; n < 8; ++n) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = warp * 16 + g4 + r * 8, j0 = n * 8 + 2 * t4;
      float pv[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int j = j0 + c;
        float d = 0.f, a = 0.f;
        if (i >= j) {
          d = i == j ? 1.f : expf((hi[i] - hi[j]) + (lo[i] - lo[j]));
          if (i > j) a = kk_acc[n][2 * r + c] * d * be[j];
          d = qk_acc[n][2 * r + c] * d * p.scale * be[j];
        }
        s_a[i * kPad + j] = a;
        s_n[i * kPad + j] = 0.f;
        pv[c] = d;
      }
      uint32_t w[NS];
      split_pair<NS>(pv[0], pv[1], w);
#pragma unroll
      for (int q = 0; q < NS; ++q)
        *reinterpret_cast<uint32_t*>(p.p_mat + mat + q * (kChunk * kChunk) + i * kChunk + j0) = w[q];
    }
  }
  __syncthreads();

  // N = (I + A)^-1.  16 x 16 blocks on the diagonal by substitution, a column
  // a lane; then [[B, 0], [C, D]]^-1 = [[B', 0], [-D' C B', D']] twice.
  if (lane < 16) {
    float x[16];
    const float* a = s_a + (warp * 16) * kPad + warp * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == lane ? 1.f : 0.f;
#pragma unroll
      for (int l = 0; l < i; ++l) v = fmaf(-a[i * kPad + l], x[l], v);
      x[i] = v;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s_n[(warp * 16 + i) * kPad + warp * 16 + lane] = x[i];
  }
  __syncthreads();
  float* s_t = s_a;  // the products C B' overwrite the blocks C that they use up
#pragma unroll
  for (int half = 16; half <= 32; half <<= 1) {
    // per 2*half block: rows half..2*half, columns 0..half.  A thread takes
    // one column and `per` rows.
    const int per = half * half * (32 / half) / kPrepThreads;  // 4, 8
    const int item = tid * per;
    const int blk = item / (half * half), in = item - blk * half * half;
    const int col = (in / per) % half, row = (in / per) / half * per;
    const int o = blk * 2 * half;
    float acc[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) acc[r] = 0.f;
    for (int l = 0; l < half; ++l) {
      const float nv = s_n[(o + l) * kPad + o + col];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < per) acc[r] = fmaf(s_a[(o + half + row + r) * kPad + o + l], nv, acc[r]);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < per) s_t[(o + half + row + r) * kPad + o + col] = acc[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r) acc[r] = 0.f;
    for (int l = 0; l < half; ++l) {
      const float tv = s_t[(o + half + l) * kPad + o + col];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < per) acc[r] = fmaf(-s_n[(o + half + row + r) * kPad + o + half + l], tv, acc[r]);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < per) s_n[(o + half + row + r) * kPad + o + col] = acc[r];
    __syncthreads();
  }

  for (int s = tid; s < kChunk * kChunk / 8; s += kPrepThreads) {
    const int i = s / (kChunk / 8), j0 = (s % (kChunk / 8)) * 8;
    uint32_t w[4][NS];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      split_pair<NS>(s_n[i * kPad + j0 + 2 * c], s_n[i * kPad + j0 + 2 * c + 1], w[c]);
#pragma unroll
    for (int q = 0; q < NS; ++q)
      *reinterpret_cast<uint4*>(p.n_mat + mat + q * (kChunk * kChunk) + i * kChunk + j0) =
          make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
  }
}

// ------------------------------------------------------------------ along the chunks
struct ScanParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  int64_t part_stride;
  const void* v;
  const __nv_bfloat16* n_mat;
  const __nv_bfloat16* p_mat;
  const float* vecs;
  const float* initial;
  float* final_state;
  void* out;                  // KEEP false
  __nv_bfloat16* e_parts;     // KEEP true
  __nv_bfloat16* s_parts;
  int64_t L, chunks;
  int key_heads, heads, dk, dv, slices;
  float scale;
};

// KEEP: no output; E and the states entering the chunks are written as parts
// (what the backward pass multiplies with).
template <typename T, int NP, int LV, int DKP, int NW, bool KEEP>
struct ScanCfg {
  static constexpr int NS = LV + 1;
  static constexpr int kTileK = kChunk * DKP * 2;
  static constexpr int kRowV = NW * 16 * (int)sizeof(T);
  static constexpr int kTileV = kChunk * kRowV;
  static constexpr int kMat = kChunk * kChunk * 2;
  static constexpr int oQ = NP * kTileK;
  static constexpr int oV = oQ + (KEEP ? 0 : NP * kTileK);
  static constexpr int oN = oV + kTileV;
  static constexpr int oP = oN + NS * kMat;
  static constexpr int oVec = oP + (KEEP ? 0 : NS * kMat);
  static constexpr int kStage = oVec + 3 * kChunk * 4 + 256;  // enter, leave, beta
  static constexpr int kStages = 2 * kStage + 128 <= 227 * 1024 ? 2 : 1;
  static constexpr int kSmem = kStages * kStage + 128;
  static_assert(kStage % 128 == 0 && kSmem <= 227 * 1024);
};

template <typename T, int NP, int LV, int DKP, int NW, bool KEEP>
__global__ void __launch_bounds__(NW * 32) delta_scan_kernel(const ScanParams p) {
  using Cfg = ScanCfg<T, NP, LV, DKP, NW, KEEP>;
  constexpr int NS = Cfg::NS, NTH = NW * 32, ROWB = DKP * 2, NT = DKP / 8;
  constexpr int MROW = kChunk * 2;  // bytes of a row of N and P
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t sm0 = smem_addr(dsm);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int64_t bh = blockIdx.x / p.slices;
  const int slice = (int)(blockIdx.x - bh * p.slices);
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int dv_cta = slice * NW * 16, dv0 = dv_cta + warp * 16;
  const int nval = p.dv - dv0;  // values of this warp's 16 rows that exist (may be <= 0)
  const int64_t kstride = (int64_t)p.key_heads * p.dk, vstride = (int64_t)p.heads * p.dv;
  const int vunits = min(NW * 16, p.dv - dv_cta) * (int)sizeof(T) / 16;

  auto load = [&](int64_t c, int s) {
    const uint32_t st = sm0 + s * Cfg::kStage;
    const int64_t t0 = c * kChunk;
    const int rows = (int)min((int64_t)kChunk, p.L - t0);
    const int64_t kf = (b * p.L + t0) * kstride + (int64_t)hk * p.dk;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      load_tile<kChunk, ROWB, NTH>(st + i * Cfg::kTileK, p.k + i * p.part_stride + kf, kstride * 2,
                                   rows, p.dk / 8, tid);
      if (!KEEP)
        load_tile<kChunk, ROWB, NTH>(st + Cfg::oQ + i * Cfg::kTileK, p.q + i * p.part_stride + kf,
                                     kstride * 2, rows, p.dk / 8, tid);
    }
    load_tile<kChunk, Cfg::kRowV, NTH>(
        st + Cfg::oV, static_cast<const T*>(p.v) + (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv_cta,
        vstride * (int)sizeof(T), rows, vunits, tid);
    const int64_t mat = (bh * p.chunks + c) * NS * (kChunk * kChunk);
    load_tile<NS * kChunk, MROW, NTH>(st + Cfg::oN, p.n_mat + mat, MROW, NS * kChunk, 8, tid);
    if (!KEEP) load_tile<NS * kChunk, MROW, NTH>(st + Cfg::oP, p.p_mat + mat, MROW, NS * kChunk, 8, tid);
    const char* vec = reinterpret_cast<const char*>(p.vecs + (bh * p.chunks + c) * (kVecCount * kChunk));
    for (int i = tid; i < 3 * kChunk * 4 / 16; i += NTH) cp16(st + Cfg::oVec + i * 16, vec + i * 16, true);
    cp_commit();
  };

  pdl_wait();
  pdl_launch_dependents();

  float S[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 4; ++c) S[n][c] = 0.f;
    if (p.initial != nullptr) {
      const int dk = n * 8 + 2 * t4;
      const float* src = p.initial + (bh * p.dv + dv0 + g4) * p.dk + dk;
      if (dk < p.dk) {
        if (g4 < nval) {
          const float2 v = *reinterpret_cast<const float2*>(src);
          S[n][0] = v.x;
          S[n][1] = v.y;
        }
        if (g4 + 8 < nval) {
          const float2 v = *reinterpret_cast<const float2*>(src + 8 * p.dk);
          S[n][2] = v.x;
          S[n][3] = v.y;
        }
      }
    }
  }

  if (Cfg::kStages == 2) load(0, 0);
  for (int64_t c = 0; c < p.chunks; ++c) {
    const int s = Cfg::kStages == 2 ? (int)(c & 1) : 0;
    if (Cfg::kStages == 1) {
      load(c, 0);
      cp_wait<0>();
    } else if (c + 1 < p.chunks) {
      load(c + 1, s ^ 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    if (nval > 0) {
      const uint32_t st = sm0 + s * Cfg::kStage;
      const float* vec = reinterpret_cast<const float*>(dsm + s * Cfg::kStage + Cfg::oVec);
      const float* enter = vec + kVecEnter * kChunk;
      const float* leave = vec + kVecLeave * kChunk;
      const float* beta = vec + kVecBeta * kChunk;
      const float total = enter[kChunk - 1];
      const int64_t t0 = c * kChunk;

      if (KEEP) {
        __nv_bfloat16* sp = p.s_parts + (bh * p.chunks + c) * NS * p.dv * DKP;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            uint32_t w[NS];
            split_pair<NS>(S[n][2 * r], S[n][2 * r + 1], w);
            if (g4 + 8 * r < nval)
#pragma unroll
              for (int q = 0; q < NS; ++q)
                *reinterpret_cast<uint32_t*>(sp + ((int64_t)q * p.dv + dv0 + g4 + 8 * r) * DKP +
                                             n * 8 + 2 * t4) = w[q];
          }
      }

      // X = (K S0^T)^T, O = (Q S0^T)^T: 16 values x 64 tokens
      float X[8][4], O[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) X[n][e] = O[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DKP / 16; ++kk) {
        uint32_t a[NS][4];
        split_frag<NS>(S[2 * kk], S[2 * kk + 1], a);
#pragma unroll
        for (int n2 = 0; n2 < 4; ++n2) {
          Step<LV == 2, 4> s;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t kb[4], qb[4];
            ldsm4(kb, at_b<ROWB>(st + i * Cfg::kTileK, lane, n2 * 16, kk));
            if (!KEEP) ldsm4(qb, at_b<ROWB>(st + Cfg::oQ + i * Cfg::kTileK, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, X[2 * n2], a[j], kb[0], kb[1]);
              s.mma(1, X[2 * n2 + 1], a[j], kb[2], kb[3]);
              if (!KEEP) {
                s.mma(2, O[2 * n2], a[j], qb[0], qb[1]);
                s.mma(3, O[2 * n2 + 1], a[j], qb[2], qb[3]);
              }
            }
          }
          s.add(0, X[2 * n2]);
          s.add(1, X[2 * n2 + 1]);
          if (!KEEP) {
            s.add(2, O[2 * n2]);
            s.add(3, O[2 * n2 + 1]);
          }
        }
      }

      // R = V - exp(G) X, in place; O *= scale exp(G)
#pragma unroll
      for (int n2 = 0; n2 < 4; ++n2) {
        uint32_t vb[4];
        if constexpr (sizeof(T) == 2) {
          const int m = lane >> 3, r = lane & 7;
          ldsm4_t(vb, tile_at<Cfg::kRowV>(st + Cfg::oV, n2 * 16 + (m >> 1) * 8 + r,
                                          warp * 2 + (m & 1)));
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int n = 2 * n2 + half, tok = n * 8 + 2 * t4;
          const float2 ge = *reinterpret_cast<const float2*>(enter + tok);
          float v[4];
          if constexpr (sizeof(T) == 2) {
            const float2 x = unpack2<T>(vb[2 * half]), y = unpack2<T>(vb[2 * half + 1]);
            v[0] = x.x;
            v[1] = x.y;
            v[2] = y.x;
            v[3] = y.y;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int row = tok + (e & 1), col = warp * 16 + g4 + (e >> 1) * 8;
              const uint32_t at = tile_at<Cfg::kRowV>(st + Cfg::oV, row, col / 4) + (col % 4) * 4;
              asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[e]) : "r"(at) : "memory");
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float w = (e & 1) ? ge.y : ge.x;
            X[n][e] = fmaf(-w, X[n][e], v[e]);
            if (!KEEP) O[n][e] *= w * p.scale;
          }
        }
      }

      // An infinity or a NaN in R (of v, k, or the state) spoils its row of
      // values from that token on, but the zeros above the diagonals of N
      // and P would carry it to earlier tokens: it is taken out here and
      // put back into E, O and the state below.
      int spoilt[2] = {kChunk, kChunk};  // first such token of the thread's two rows
      float probe = 0.f;
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) probe = fmaf(X[n][e], 0.f, probe);
      const bool bad = __any_sync(0xffffffffu, probe != 0.f);
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
      auto spoil = [&](float (&y)[8][4]) {
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n * 8 + 2 * t4 + (e & 1) >= spoilt[e >> 1]) y[n][e] = __int_as_float(0x7fc00000);
      };

      // E = N R
      float E[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) E[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t a[NS][4];
        split_frag<NS>(X[2 * kk], X[2 * kk + 1], a);
#pragma unroll
        for (int n2 = kk; n2 < 4; ++n2) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int i = LV; i >= 0; --i) {
            uint32_t nb[4];
            ldsm4(nb, at_b<MROW>(st + Cfg::oN + i * Cfg::kMat, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, E[2 * n2], a[j], nb[0], nb[1]);
              s.mma(1, E[2 * n2 + 1], a[j], nb[2], nb[3]);
            }
          }
          s.add(0, E[2 * n2]);
          s.add(1, E[2 * n2 + 1]);
        }
      }

      if (KEEP) {
        if (bad) spoil(E);
        __nv_bfloat16* ep = p.e_parts + (bh * p.chunks + c) * NS * kChunk * p.dv + dv0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          uint32_t lo[NS], hi[NS];
          split_pair<NS>(E[n][0], E[n][1], lo);
          split_pair<NS>(E[n][2], E[n][3], hi);
#pragma unroll
          for (int q = 0; q < NS; ++q) {
            const uint32_t x = movmatrix_t(lo[q]), y = movmatrix_t(hi[q]);
            __nv_bfloat16* o = ep + ((int64_t)q * kChunk + n * 8 + g4) * p.dv + 2 * t4;
            *reinterpret_cast<uint32_t*>(o) = x;
            if (nval > 8) *reinterpret_cast<uint32_t*>(o + 8) = y;
          }
        }
      } else {
        // O += P E
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t a[NS][4];
          split_frag<NS>(E[2 * kk], E[2 * kk + 1], a);
#pragma unroll
          for (int n2 = kk; n2 < 4; ++n2) {
            Step<LV == 2, 2> s;
#pragma unroll
            for (int i = LV; i >= 0; --i) {
              uint32_t pb[4];
              ldsm4(pb, at_b<MROW>(st + Cfg::oP + i * Cfg::kMat, lane, n2 * 16, kk));
#pragma unroll
              for (int j = LV - i; j >= 0; --j) {
                s.mma(0, O[2 * n2], a[j], pb[0], pb[1]);
                s.mma(1, O[2 * n2 + 1], a[j], pb[2], pb[3]);
              }
            }
            s.add(0, O[2 * n2]);
            s.add(1, O[2 * n2 + 1]);
          }
        }
        T* out = static_cast<T*>(p.out) + (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv0;
        const int rows = (int)min((int64_t)kChunk, p.L - t0);
        if (bad) spoil(O);
#pragma unroll
        for (int n = 0; n < 8; ++n)
          store_t<T>(out + (int64_t)n * 8 * vstride, vstride, O[n], lane, rows - n * 8, nval);
      }

      // S = exp(G_C) S + (beta exp(G_C - G) E)^T K.  The chunk's sum starts
      // at zero and joins the state in one rounded multiply-add.
      uint32_t u[4][NS][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int tok = (2 * kk + half) * 8 + 2 * t4;
          const float2 lv = *reinterpret_cast<const float2*>(leave + tok);
          const float2 bt = *reinterpret_cast<const float2*>(beta + tok);
          const float w0 = lv.x * bt.x, w1 = lv.y * bt.y;
          E[2 * kk + half][0] *= w0;
          E[2 * kk + half][1] *= w1;
          E[2 * kk + half][2] *= w0;
          E[2 * kk + half][3] *= w1;
        }
        split_frag<NS>(E[2 * kk], E[2 * kk + 1], u[kk]);
      }
#pragma unroll
      for (int n4 = 0; n4 < NT / 4; ++n4) {
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
            ldsm4_t(b0, at_bt<ROWB>(st + i * Cfg::kTileK, lane, n4 * 32, kk));
            ldsm4_t(b1, at_bt<ROWB>(st + i * Cfg::kTileK, lane, n4 * 32 + 16, kk));
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
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (spoilt[e >> 1] < kChunk) S[n][e] = __int_as_float(0x7fc00000);
    }
    __syncthreads();
  }

  if (p.final_state != nullptr && nval > 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int dk = n * 8 + 2 * t4;
      float* dst = p.final_state + (bh * p.dv + dv0 + g4) * p.dk + dk;
      if (dk < p.dk) {
        if (g4 < nval) *reinterpret_cast<float2*>(dst) = make_float2(S[n][0], S[n][1]);
        if (g4 + 8 < nval)
          *reinterpret_cast<float2*>(dst + 8 * p.dk) = make_float2(S[n][2], S[n][3]);
      }
    }
  }
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
  return launch_pdl(kern, (unsigned)(bh * p.slices), NW * 32, Cfg::kSmem, a.stream, p);
}

}  // namespace

// Prep and scan for sequences [b0, b0 + nb) of the call.  keep: for the
// backward pass (E and the states instead of the output).
template <typename T, int LV, int DKP>
cudaError_t delta_fwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb,
                           bool keep) {
  constexpr int NP = kParts<T>;
  char* ws = static_cast<char*>(a.workspace);
  const int64_t nk = nb * a.seqlen * a.key_heads * a.dk, nv = nb * a.seqlen * a.heads * a.dv;
  const int64_t k0 = b0 * a.seqlen * a.key_heads * a.dk, v0 = b0 * a.seqlen * a.heads * a.dv;
  const int64_t g0 = b0 * a.seqlen * a.heads, s0 = b0 * a.heads * a.dv * a.dk;
  const T* q = static_cast<const T*>(a.q) + k0;
  const T* k = static_cast<const T*>(a.k) + k0;
  PrepParams pp{};
  if constexpr (NP > 1) {
    SplitParams sp{};
    sp.src[0] = q;
    sp.src[1] = k;
    sp.dst[0] = reinterpret_cast<__nv_bfloat16*>(ws + pl.q_parts);
    sp.dst[1] = reinterpret_cast<__nv_bfloat16*>(ws + pl.k_parts);
    sp.n[0] = sp.n[1] = nk;
    if (keep) {
      sp.src[2] = static_cast<const T*>(a.grad_out) + v0;
      sp.dst[2] = reinterpret_cast<__nv_bfloat16*>(ws + pl.do_parts);
      sp.n[2] = nv;
    }
    const int64_t per = (std::max(nk, keep ? nv : 0) + 2047) / 2048;
    const unsigned grid = 3 * (unsigned)std::min<int64_t>(per, 4 * a.num_sms);
    const cudaError_t e = launch_pdl(delta_split_kernel<T>, grid, 256, 0, a.stream, sp);
    if (e != cudaSuccess) return e;
    pp.q = sp.dst[0];
    pp.k = sp.dst[1];
    pp.part_stride = nk;
  } else {
    pp.q = reinterpret_cast<const __nv_bfloat16*>(q);
    pp.k = reinterpret_cast<const __nv_bfloat16*>(k);
  }
  pp.log_decay = static_cast<const T*>(a.log_decay) + g0;
  pp.beta = static_cast<const T*>(a.beta) + g0;
  pp.n_mat = reinterpret_cast<__nv_bfloat16*>(ws + pl.n_mat);
  pp.p_mat = reinterpret_cast<__nv_bfloat16*>(ws + pl.p_mat);
  pp.vecs = reinterpret_cast<float*>(ws + pl.vecs);
  pp.L = a.seqlen;
  pp.chunks = pl.chunks;
  pp.key_heads = (int)a.key_heads;
  pp.heads = (int)a.heads;
  pp.dk = (int)a.dk;
  pp.scale = a.scale;
  const int64_t bh = nb * a.heads;
  auto prep = delta_prep_kernel<T, NP, LV, DKP>;
  cudaError_t e = configure(prep, prep_smem<NP, DKP>());
  if (e != cudaSuccess) return e;
  e = launch_pdl(prep, (unsigned)(bh * pl.chunks), kPrepThreads, prep_smem<NP, DKP>(), a.stream, pp);
  if (e != cudaSuccess) return e;

  ScanParams p{};
  p.q = pp.q;
  p.k = pp.k;
  p.part_stride = pp.part_stride;
  p.v = static_cast<const T*>(a.v) + v0;
  p.n_mat = pp.n_mat;
  p.p_mat = pp.p_mat;
  p.vecs = pp.vecs;
  p.initial = a.initial ? a.initial + s0 : nullptr;
  p.final_state = !keep && a.final_state ? a.final_state + s0 : nullptr;
  p.out = keep ? nullptr : static_cast<T*>(a.out) + v0;
  p.e_parts = reinterpret_cast<__nv_bfloat16*>(ws + pl.e_parts);
  p.s_parts = reinterpret_cast<__nv_bfloat16*>(ws + pl.s_parts);
  p.L = a.seqlen;
  p.chunks = pl.chunks;
  p.key_heads = (int)a.key_heads;
  p.heads = (int)a.heads;
  p.dk = (int)a.dk;
  p.dv = (int)a.dv;
  p.scale = a.scale;
  const bool narrow = bh * ((a.dv + 127) / 128) < a.num_sms || a.dv <= 64;
  if (keep)
    return narrow ? scan_nw<T, LV, DKP, 4, true>(a, p, bh) : scan_nw<T, LV, DKP, 8, true>(a, p, bh);
  return narrow ? scan_nw<T, LV, DKP, 4, false>(a, p, bh) : scan_nw<T, LV, DKP, 8, false>(a, p, bh);
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
    if (pl.np > 1) {
      pl.q_parts = take(pl.np * tok * key_heads * dk * 2);
      pl.k_parts = take(pl.np * tok * key_heads * dk * 2);
    }
    pl.n_mat = take(c * pl.ns * kChunk * kChunk * 2);
    pl.p_mat = take(c * pl.ns * kChunk * kChunk * 2);
    pl.vecs = take(c * kVecCount * kChunk * 4);
    if (backward) {
      if (pl.np > 1) pl.do_parts = take(pl.np * tok * heads * dv * 2);
      pl.e_parts = take(c * pl.ns * kChunk * dv * 2);
      pl.dv_parts = take(c * pl.ns * kChunk * dv * 2);
      pl.s_parts = take(c * pl.ns * dv * pl.dkp * 2);
      pl.ds_parts = take(c * pl.ns * dv * pl.dkp * 2);
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
