// Gated delta rule, backward (sm_100a).  With the chunk's N, P, E, S0 of
// delta.cuh (recomputed by the forward kernels from the inputs) and dS the
// gradient of the state leaving the chunk:
//     F  = P^T dO + beta exp(G_C - G) K dS^T,    dV = N^T F,
//     dS0 = exp(G_C) dS + scale (exp(G) dO)^T Q - (exp(G) dV)^T K      (sequential)
// and then, for every chunk by itself, with H = tril(dO E^T), X = tril(dV E^T, -1),
// Hs = scale D H, Xd = D X:
//     dQ = scale exp(G) dO S0 + Hs diag(beta) K,
//     dK = diag(beta) W + R,  R = -exp(G) dV S0 - Xd diag(beta) K,
//          W = Hs^T Q - Xd^T K + exp(G_C - G) E dS,
//     dbeta_i = k_i . W_i,
//     dlog_decay_t = sum_{i >= t} (q_i.dQ_i + k_i.R_i - beta_i dbeta_i) + <S_C, dS>.
// The last two hold because beta and k scale a write alike, and because a
// decay scales what is read after it like q and k do: no quotient of a
// gradient by beta or by a decay appears, so zeros of both are harmless.
//
//   delta_rev_kernel    from the last chunk to the first, dS^T in registers
//                       as delta_scan_kernel keeps S^T; writes dV, dS per chunk.
//   delta_grad_kernel   one CTA per (chunk, head), all in parallel.
//   delta_group_kernel  sums dQ, dK over the heads that share a key head, in
//                       a fixed order.
#include <algorithm>

#include "delta.cuh"
#include "internal.h"

namespace fpscan {

template <typename T, int LV, int DKP>
cudaError_t delta_fwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb,
                           bool keep);

namespace {

// ------------------------------------------------------------------ along the chunks, backwards
struct RevParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* grad;  // dO parts
  int64_t part_stride, grad_stride;
  const __nv_bfloat16* n_mat;
  const __nv_bfloat16* p_mat;
  const float* vecs;
  const float* grad_final;
  float* dinitial;
  void* dv_out;
  __nv_bfloat16* dv_parts;
  __nv_bfloat16* ds_parts;
  int64_t L, chunks;
  int key_heads, heads, dk, dv, slices;
  float scale;
};

template <int NP, int LV, int DKP, int NW>
struct RevCfg {
  static constexpr int NS = LV + 1;
  static constexpr int kTileK = kChunk * DKP * 2;
  static constexpr int kRowG = NW * 32;
  static constexpr int kTileG = kChunk * kRowG;
  static constexpr int kMat = kChunk * kChunk * 2;
  static constexpr int oQ = NP * kTileK;
  static constexpr int oG = oQ + NP * kTileK;
  static constexpr int oN = oG + NP * kTileG;
  static constexpr int oP = oN + NS * kMat;
  static constexpr int oVec = oP + NS * kMat;
  static constexpr int kStage = oVec + 3 * kChunk * 4 + 256;
  static constexpr int kStages = 2 * kStage + 128 <= 227 * 1024 ? 2 : 1;
  static constexpr int kSmem = kStages * kStage + 128;
  static_assert(kStage % 128 == 0 && kSmem <= 227 * 1024);
};

template <typename T, int NP, int LV, int DKP, int NW>
__global__ void __launch_bounds__(NW * 32) delta_rev_kernel(const RevParams p) {
  using Cfg = RevCfg<NP, LV, DKP, NW>;
  constexpr int NS = Cfg::NS, NTH = NW * 32, ROWB = DKP * 2, NT = DKP / 8, MROW = kChunk * 2;
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
  const int nval = p.dv - dv0;
  const int64_t kstride = (int64_t)p.key_heads * p.dk, vstride = (int64_t)p.heads * p.dv;
  const int vunits = min(NW * 16, p.dv - dv_cta) / 8;

  auto load = [&](int64_t c, int s) {
    const uint32_t st = sm0 + s * Cfg::kStage;
    const int64_t t0 = c * kChunk;
    const int rows = (int)min((int64_t)kChunk, p.L - t0);
    const int64_t kf = (b * p.L + t0) * kstride + (int64_t)hk * p.dk;
    const int64_t vf = (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv_cta;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      load_tile<kChunk, ROWB, NTH>(st + i * Cfg::kTileK, p.k + i * p.part_stride + kf, kstride * 2,
                                   rows, p.dk / 8, tid);
      load_tile<kChunk, ROWB, NTH>(st + Cfg::oQ + i * Cfg::kTileK, p.q + i * p.part_stride + kf,
                                   kstride * 2, rows, p.dk / 8, tid);
      load_tile<kChunk, Cfg::kRowG, NTH>(st + Cfg::oG + i * Cfg::kTileG,
                                         p.grad + i * p.grad_stride + vf, vstride * 2, rows, vunits,
                                         tid);
    }
    const int64_t mat = (bh * p.chunks + c) * NS * (kChunk * kChunk);
    load_tile<NS * kChunk, MROW, NTH>(st + Cfg::oN, p.n_mat + mat, MROW, NS * kChunk, 8, tid);
    load_tile<NS * kChunk, MROW, NTH>(st + Cfg::oP, p.p_mat + mat, MROW, NS * kChunk, 8, tid);
    const char* vec = reinterpret_cast<const char*>(p.vecs + (bh * p.chunks + c) * (kVecCount * kChunk));
    for (int i = tid; i < 3 * kChunk * 4 / 16; i += NTH) cp16(st + Cfg::oVec + i * 16, vec + i * 16, true);
    cp_commit();
  };

  pdl_wait();
  pdl_launch_dependents();

  float S[NT][4];  // dS^T
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 4; ++c) S[n][c] = 0.f;
    if (p.grad_final != nullptr) {
      const int dk = n * 8 + 2 * t4;
      const float* src = p.grad_final + (bh * p.dv + dv0 + g4) * p.dk + dk;
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

  if (Cfg::kStages == 2) load(p.chunks - 1, 0);
  for (int64_t done = 0; done < p.chunks; ++done) {
    const int64_t c = p.chunks - 1 - done;
    const int s = Cfg::kStages == 2 ? (int)(done & 1) : 0;
    if (Cfg::kStages == 1) {
      load(c, 0);
      cp_wait<0>();
    } else if (c > 0) {
      load(c - 1, s ^ 1);
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

      __nv_bfloat16* sp = p.ds_parts + (bh * p.chunks + c) * NS * p.dv * DKP;
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

      // Y = (K dS^T)^T, Z = (P^T dO)^T: 16 values x 64 tokens
      float Y[8][4], Z[8][4];
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) Y[n][e] = Z[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < DKP / 16; ++kk) {
        uint32_t a[NS][4];
        split_frag<NS>(S[2 * kk], S[2 * kk + 1], a);
#pragma unroll
        for (int n2 = 0; n2 < 4; ++n2) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t kb[4];
            ldsm4(kb, at_b<ROWB>(st + i * Cfg::kTileK, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, Y[2 * n2], a[j], kb[0], kb[1]);
              s.mma(1, Y[2 * n2 + 1], a[j], kb[2], kb[3]);
            }
          }
          s.add(0, Y[2 * n2]);
          s.add(1, Y[2 * n2 + 1]);
        }
      }
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t a[NP][4];
#pragma unroll
        for (int i = 0; i < NP; ++i)
          ldsm4_t(a[i], at_at<Cfg::kRowG>(st + Cfg::oG + i * Cfg::kTileG, lane, warp * 16, kk));
#pragma unroll
        for (int n2 = 0; n2 <= kk; ++n2) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int j = LV; j >= 0; --j) {
            uint32_t pb[4];
            ldsm4_t(pb, at_bt<MROW>(st + Cfg::oP + j * Cfg::kMat, lane, n2 * 16, kk));
#pragma unroll
            for (int i = NP - 1; i >= 0; --i) {
              if (i + j > LV) continue;
              s.mma(0, Z[2 * n2], a[i], pb[0], pb[1]);
              s.mma(1, Z[2 * n2 + 1], a[i], pb[2], pb[3]);
            }
          }
          s.add(0, Z[2 * n2]);
          s.add(1, Z[2 * n2 + 1]);
        }
      }
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int tok = n * 8 + 2 * t4;
        const float2 lv = *reinterpret_cast<const float2*>(leave + tok);
        const float2 bt = *reinterpret_cast<const float2*>(beta + tok);
        const float w0 = lv.x * bt.x, w1 = lv.y * bt.y;
        Z[n][0] = fmaf(w0, Y[n][0], Z[n][0]);
        Z[n][1] = fmaf(w1, Y[n][1], Z[n][1]);
        Z[n][2] = fmaf(w0, Y[n][2], Z[n][2]);
        Z[n][3] = fmaf(w1, Y[n][3], Z[n][3]);
      }

      // dV = N^T F (in Y)
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) Y[n][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        uint32_t a[NS][4];
        split_frag<NS>(Z[2 * kk], Z[2 * kk + 1], a);
#pragma unroll
        for (int n2 = 0; n2 <= kk; ++n2) {
          Step<LV == 2, 2> s;
#pragma unroll
          for (int i = LV; i >= 0; --i) {
            uint32_t nb[4];
            ldsm4_t(nb, at_bt<MROW>(st + Cfg::oN + i * Cfg::kMat, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, Y[2 * n2], a[j], nb[0], nb[1]);
              s.mma(1, Y[2 * n2 + 1], a[j], nb[2], nb[3]);
            }
          }
          s.add(0, Y[2 * n2]);
          s.add(1, Y[2 * n2 + 1]);
        }
      }
      {
        T* out = static_cast<T*>(p.dv_out) + (b * p.L + t0) * vstride + (int64_t)h * p.dv + dv0;
        const int rows = (int)min((int64_t)kChunk, p.L - t0);
        __nv_bfloat16* vp = p.dv_parts + (bh * p.chunks + c) * NS * kChunk * p.dv + dv0;
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          store_t<T>(out + (int64_t)n * 8 * vstride, vstride, Y[n], lane, rows - n * 8, nval);
          uint32_t lo[NS], hi[NS];
          split_pair<NS>(Y[n][0], Y[n][1], lo);
          split_pair<NS>(Y[n][2], Y[n][3], hi);
#pragma unroll
          for (int q = 0; q < NS; ++q) {
            const uint32_t x = movmatrix_t(lo[q]), y = movmatrix_t(hi[q]);
            __nv_bfloat16* o = vp + ((int64_t)q * kChunk + n * 8 + g4) * p.dv + 2 * t4;
            *reinterpret_cast<uint32_t*>(o) = x;
            if (nval > 8) *reinterpret_cast<uint32_t*>(o + 8) = y;
          }
        }
      }

      // dS <- exp(G_C) dS + (scale exp(G) dO)^T Q - (exp(G) dV)^T K
      uint32_t ug[4][NS][4], uv[4][NS][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        float x[4][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r][0] = x[r][1] = 0.f;
#pragma unroll
        for (int i = NP - 1; i >= 0; --i) {
          uint32_t a[4];
          ldsm4_t(a, at_at<Cfg::kRowG>(st + Cfg::oG + i * Cfg::kTileG, lane, warp * 16, kk));
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[r][0] += bf16_lo(a[r]);
            x[r][1] += bf16_hi(a[r]);
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float2 ge = *reinterpret_cast<const float2*>(enter + kk * 16 + half * 8 + 2 * t4);
          const int n = 2 * kk + half;
          Y[n][0] *= -ge.x;
          Y[n][1] *= -ge.y;
          Y[n][2] *= -ge.x;
          Y[n][3] *= -ge.y;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            x[2 * half + r][0] *= ge.x * p.scale;
            x[2 * half + r][1] *= ge.y * p.scale;
            uint32_t w[NS];
            split_pair<NS>(x[2 * half + r][0], x[2 * half + r][1], w);
#pragma unroll
            for (int q = 0; q < NS; ++q) ug[kk][q][2 * half + r] = w[q];
          }
        }
        split_frag<NS>(Y[2 * kk], Y[2 * kk + 1], uv[kk]);
      }
#pragma unroll
      for (int n2 = 0; n2 < NT / 2; ++n2) {
        float d[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          Step<LV == 2, 4> s;
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) {
            uint32_t qb[4], kb[4];
            ldsm4_t(qb, at_bt<ROWB>(st + Cfg::oQ + i * Cfg::kTileK, lane, n2 * 16, kk));
            ldsm4_t(kb, at_bt<ROWB>(st + i * Cfg::kTileK, lane, n2 * 16, kk));
#pragma unroll
            for (int j = LV - i; j >= 0; --j) {
              s.mma(0, d[0], ug[kk][j], qb[0], qb[1]);
              s.mma(1, d[1], ug[kk][j], qb[2], qb[3]);
              s.mma(2, d[0], uv[kk][j], kb[0], kb[1]);
              s.mma(3, d[1], uv[kk][j], kb[2], kb[3]);
            }
          }
#pragma unroll
          for (int n = 0; n < 4; ++n) s.add(n, d[n & 1]);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[n2 * 2 + n][e] = fmaf(total, S[n2 * 2 + n][e], d[n][e]);
      }
    }
    __syncthreads();
  }

  if (p.dinitial != nullptr && nval > 0) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int dk = n * 8 + 2 * t4;
      float* dst = p.dinitial + (bh * p.dv + dv0 + g4) * p.dk + dk;
      if (dk < p.dk) {
        if (g4 < nval) *reinterpret_cast<float2*>(dst) = make_float2(S[n][0], S[n][1]);
        if (g4 + 8 < nval)
          *reinterpret_cast<float2*>(dst + 8 * p.dk) = make_float2(S[n][2], S[n][3]);
      }
    }
  }
}

// ------------------------------------------------------------------ gradients of a chunk
struct GradParams {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* grad;
  int64_t part_stride, grad_stride;
  const __nv_bfloat16* e_parts;
  const __nv_bfloat16* dv_parts;
  const __nv_bfloat16* s_parts;
  const __nv_bfloat16* ds_parts;
  const float* vecs;
  const void* log_decay;
  void* dq;              // T (batch, seqlen, key_heads, dk), or nullptr:
  void* dk_out;
  float* dq_part;        // fp32 (batch, seqlen, heads, dk), summed afterwards
  float* dk_part;
  void* dlog_decay;
  void* dbeta;
  int64_t L, chunks;
  int key_heads, heads, dk, dv;
  float scale;
};

constexpr int kGradThreads = 256;
constexpr int kSlice = 64;  // values (dv) per step of the first phase

template <int NP, int LV, int DKP>
struct GradCfg {
  static constexpr int NS = LV + 1;
  static constexpr int kTileK = kChunk * DKP * 2;
  static constexpr int kTileV = kChunk * kSlice * 2;
  static constexpr int kMat = kChunk * kChunk * 2;
  // first phase: dO, dV, E, S0, dS of one slice
  static constexpr int oV = NP * kTileV;
  static constexpr int oE = oV + NS * kTileV;
  static constexpr int oS = oE + NS * kTileV;
  static constexpr int oD = oS + NS * kSlice * DKP * 2;
  static constexpr int kFirst = oD + NS * kSlice * DKP * 2;
  // second phase, over the first's: K, Q, and four matrices
  static constexpr int oQ = NP * kTileK;
  static constexpr int oHs = 2 * NP * kTileK;
  static constexpr int oHb = oHs + NS * kMat;
  static constexpr int oXd = oHb + NS * kMat;
  static constexpr int oXb = oXd + NS * kMat;
  static constexpr int kSecond = oXb + NS * kMat;
  static constexpr int kBody = kFirst > kSecond ? kFirst : kSecond;
  static constexpr int kSmem = kBody + 128;
  static_assert(kSmem + 8192 <= 227 * 1024);
};

template <typename T, int NP, int LV, int DKP>
__global__ void __launch_bounds__(kGradThreads, 1) delta_grad_kernel(const GradParams p) {
  using Cfg = GradCfg<NP, LV, DKP>;
  constexpr int NS = Cfg::NS, NTH = kGradThreads, ROWB = DKP * 2, VROW = kSlice * 2, MROW = kChunk * 2;
  constexpr int NT = DKP / 32;  // n tiles of a warp's DKP / 4 columns
  extern __shared__ __align__(128) unsigned char dsm_raw[];
  unsigned char* dsm = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(dsm_raw) + 127) & ~uintptr_t(127));
  const uint32_t st = smem_addr(dsm);
  __shared__ __align__(16) float s_vec[kVecCount * kChunk];
  __shared__ float s_red[3][4][kChunk];
  __shared__ float s_dot[NTH / 32];

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, t4 = lane & 3;
  const int wr = warp >> 2, wc = warp & 3;
  const int64_t bh = blockIdx.x / p.chunks, chunk = blockIdx.x - bh * p.chunks;
  const int64_t b = bh / p.heads;
  const int h = (int)(bh - b * p.heads), hk = h / (p.heads / p.key_heads);
  const int64_t t0 = chunk * kChunk;
  const int rows = (int)min((int64_t)kChunk, p.L - t0);
  const int64_t kstride = (int64_t)p.key_heads * p.dk, vstride = (int64_t)p.heads * p.dv;
  const int64_t kf = (b * p.L + t0) * kstride + (int64_t)hk * p.dk;
  const int64_t unit = bh * p.chunks + chunk;

  pdl_wait();
  pdl_launch_dependents();
  {
    const char* vec = reinterpret_cast<const char*>(p.vecs + unit * (kVecCount * kChunk));
    const uint32_t dst = smem_addr(s_vec);
    for (int i = tid; i < kVecCount * kChunk * 4 / 16; i += NTH) cp16(dst + i * 16, vec + i * 16, true);
  }

  float aq[2][NT][4], ar[2][NT][4], aw[2][NT][4], ah[2][2][4], ax[2][2][4];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) aq[m][n][e] = ar[m][n][e] = aw[m][n][e] = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) ah[m][n][e] = ax[m][n][e] = 0.f;
  }
  const bool lower = wc * 16 <= wr * 32 + 31;  // this warp's tile of H and X reaches the lower triangle
  const int col0 = wc * (DKP / 4);
  float dot = 0.f;  // this thread's share of <S0, dS>

  for (int v0 = 0; v0 < p.dv; v0 += kSlice) {
    const int vals = min(kSlice, p.dv - v0);
    const int64_t vf = (b * p.L + t0) * vstride + (int64_t)h * p.dv + v0;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      load_tile<kChunk, VROW, NTH>(st + i * Cfg::kTileV, p.grad + i * p.grad_stride + vf,
                                   vstride * 2, rows, vals / 8, tid);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int64_t ev = (unit * NS + i) * kChunk * p.dv + v0;
      const int64_t sv = ((unit * NS + i) * p.dv + v0) * DKP;
      load_tile<kChunk, VROW, NTH>(st + Cfg::oV + i * Cfg::kTileV, p.dv_parts + ev, (int64_t)p.dv * 2,
                                   kChunk, vals / 8, tid);
      load_tile<kChunk, VROW, NTH>(st + Cfg::oE + i * Cfg::kTileV, p.e_parts + ev, (int64_t)p.dv * 2,
                                   kChunk, vals / 8, tid);
      load_tile<kSlice, ROWB, NTH>(st + Cfg::oS + i * kSlice * ROWB, p.s_parts + sv, ROWB, vals,
                                   ROWB / 16, tid);
      load_tile<kSlice, ROWB, NTH>(st + Cfg::oD + i * kSlice * ROWB, p.ds_parts + sv, ROWB, vals,
                                   ROWB / 16, tid);
    }
    cp_commit();
    cp_wait<0>();
    __syncthreads();

#pragma unroll
    for (int kk = 0; kk < kSlice / 16; ++kk) {
      {
        uint32_t ag[NP][2][4], av[NS][2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
          for (int i = 0; i < NP; ++i)
            ldsm4(ag[i][m], at_a<VROW>(st + i * Cfg::kTileV, lane, wr * 32 + m * 16, kk));
#pragma unroll
          for (int i = 0; i < NS; ++i)
            ldsm4(av[i][m], at_a<VROW>(st + Cfg::oV + i * Cfg::kTileV, lane, wr * 32 + m * 16, kk));
        }
        if (lower) {
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            Step<LV == 2, 4> s;
#pragma unroll
            for (int j = LV; j >= 0; --j) {
              uint32_t eb[4];
              ldsm4(eb, at_b<VROW>(st + Cfg::oE + j * Cfg::kTileV, lane, wc * 16, kk));
#pragma unroll
              for (int i = LV - j; i >= 0; --i) {
                if (i < NP) {
                  s.mma(0, ah[m][0], ag[i < NP ? i : 0][m], eb[0], eb[1]);
                  s.mma(1, ah[m][1], ag[i < NP ? i : 0][m], eb[2], eb[3]);
                }
                s.mma(2, ax[m][0], av[i][m], eb[0], eb[1]);
                s.mma(3, ax[m][1], av[i][m], eb[2], eb[3]);
              }
            }
            s.add(0, ah[m][0]);
            s.add(1, ah[m][1]);
            s.add(2, ax[m][0]);
            s.add(3, ax[m][1]);
          }
        }
#pragma unroll
        for (int n2 = 0; n2 < NT / 2; ++n2) {
          Step<LV == 2, 8> s;
#pragma unroll
          for (int j = LV; j >= 0; --j) {
            uint32_t sb[4];
            ldsm4_t(sb, at_bt<ROWB>(st + Cfg::oS + j * kSlice * ROWB, lane, col0 + n2 * 16, kk));
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int i = LV - j; i >= 0; --i) {
                if (i < NP) {
                  s.mma(4 * m, aq[m][2 * n2], ag[i < NP ? i : 0][m], sb[0], sb[1]);
                  s.mma(4 * m + 1, aq[m][2 * n2 + 1], ag[i < NP ? i : 0][m], sb[2], sb[3]);
                }
                s.mma(4 * m + 2, ar[m][2 * n2], av[i][m], sb[0], sb[1]);
                s.mma(4 * m + 3, ar[m][2 * n2 + 1], av[i][m], sb[2], sb[3]);
              }
          }
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            s.add(4 * m, aq[m][2 * n2]);
            s.add(4 * m + 1, aq[m][2 * n2 + 1]);
            s.add(4 * m + 2, ar[m][2 * n2]);
            s.add(4 * m + 3, ar[m][2 * n2 + 1]);
          }
        }
      }
      uint32_t ae[NS][2][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int i = 0; i < NS; ++i)
          ldsm4(ae[i][m], at_a<VROW>(st + Cfg::oE + i * Cfg::kTileV, lane, wr * 32 + m * 16, kk));
#pragma unroll
      for (int n2 = 0; n2 < NT / 2; ++n2) {
        Step<LV == 2, 4> s;
#pragma unroll
        for (int j = LV; j >= 0; --j) {
          uint32_t db[4];
          ldsm4_t(db, at_bt<ROWB>(st + Cfg::oD + j * kSlice * ROWB, lane, col0 + n2 * 16, kk));
#pragma unroll
          for (int i = LV - j; i >= 0; --i)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              s.mma(2 * m, aw[m][2 * n2], ae[i][m], db[0], db[1]);
              s.mma(2 * m + 1, aw[m][2 * n2 + 1], ae[i][m], db[2], db[3]);
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          s.add(2 * m, aw[m][2 * n2]);
          s.add(2 * m + 1, aw[m][2 * n2 + 1]);
        }
      }
    }
    // <S0, dS> over this slice (the same place of every part: swizzle does not matter)
    for (int i = tid; i < kSlice * DKP / 2; i += NTH) {
      float x0 = 0.f, x1 = 0.f, y0 = 0.f, y1 = 0.f;
#pragma unroll
      for (int q = NS - 1; q >= 0; --q) {
        const uint32_t x = *reinterpret_cast<const uint32_t*>(dsm + Cfg::oS + q * kSlice * ROWB + i * 4);
        const uint32_t y = *reinterpret_cast<const uint32_t*>(dsm + Cfg::oD + q * kSlice * ROWB + i * 4);
        x0 += bf16_lo(x);
        x1 += bf16_hi(x);
        y0 += bf16_lo(y);
        y1 += bf16_hi(y);
      }
      dot = fmaf(x0, y0, fmaf(x1, y1, dot));
    }
    __syncthreads();
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
  if (lane == 0) s_dot[warp] = dot;

  // second phase: K and Q take the place of the slices
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    load_tile<kChunk, ROWB, NTH>(st + i * Cfg::kTileK, p.k + i * p.part_stride + kf, kstride * 2, rows,
                                 p.dk / 8, tid);
    load_tile<kChunk, ROWB, NTH>(st + Cfg::oQ + i * Cfg::kTileK, p.q + i * p.part_stride + kf,
                                 kstride * 2, rows, p.dk / 8, tid);
  }
  cp_commit();
  const float* enter = s_vec + kVecEnter * kChunk;
  const float* leave = s_vec + kVecLeave * kChunk;
  const float* beta = s_vec + kVecBeta * kChunk;
  const float* hi = s_vec + kVecCumHi * kChunk;
  const float* lo = s_vec + kVecCumLo * kChunk;
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int i = wr * 32 + m * 16 + r * 8 + g4, j0 = wc * 16 + n * 8 + 2 * t4;
        float hs[2], hb[2], xd[2], xb[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int j = j0 + c;
          hs[c] = xd[c] = 0.f;
          if (i >= j) {
            const float d = i == j ? 1.f : expf((hi[i] - hi[j]) + (lo[i] - lo[j]));
            hs[c] = ah[m][n][2 * r + c] * d * p.scale;
            if (i > j) xd[c] = -ax[m][n][2 * r + c] * d;
          }
          hb[c] = hs[c] * beta[j];
          xb[c] = xd[c] * beta[j];
        }
        const uint32_t at = tile_at<MROW>(0, i, j0 / 8) + (j0 % 8) * 2;
        uint32_t w[NS];
        auto put = [&](const float* x, int off) {
          split_pair<NS>(x[0], x[1], w);
#pragma unroll
          for (int q = 0; q < NS; ++q)
            *reinterpret_cast<uint32_t*>(dsm + off + q * Cfg::kMat + at) = w[q];
        };
        put(hs, Cfg::oHs);
        put(hb, Cfg::oHb);
        put(xd, Cfg::oXd);
        put(xb, Cfg::oXb);
      }
  cp_wait<0>();
  __syncthreads();

  // an element pair of K or Q as fp32 (the sum of its parts)
  auto kq_pair = [&](int off, int row, int col) {
    float2 v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = NP - 1; i >= 0; --i) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(
          dsm + off + i * Cfg::kTileK + tile_at<ROWB>(0, row, col / 8) + (col % 8) * 2);
      v.x += bf16_lo(w);
      v.y += bf16_hi(w);
    }
    return v;
  };
  // sums over a warp's columns of a row, one value per row and warp column
  auto put_row = [&](int which, int row, float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    v += __shfl_xor_sync(0xffffffffu, v, 2);
    if (t4 == 0) s_red[which][wc][row] = v;
  };
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = wr * 32 + m * 16 + r * 8 + g4;
      const float ge = enter[i], gl = leave[i];
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 kv = kq_pair(0, i, col0 + n * 8 + 2 * t4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          aq[m][n][2 * r + c] *= ge * p.scale;
          ar[m][n][2 * r + c] *= -ge;
          aw[m][n][2 * r + c] *= gl;
          sum = fmaf(aw[m][n][2 * r + c], c ? kv.y : kv.x, sum);
        }
      }
      put_row(2, i, sum);
    }

#pragma unroll
  for (int kk = 0; kk < 4; ++kk) {
    const bool left = kk <= 2 * wr + 1;   // columns j = 16 kk.. of rows i: j <= i somewhere
    const bool right = kk >= 2 * wr;      // rows i = 16 kk.. of columns j: i >= j somewhere
    // the matrices' parts i and K's or Q's parts j, smallest first
    auto product = [&](int hs, int xs, bool trans, int hb_off, float (&h_acc)[2][NT][4],
                       float (&x_acc)[2][NT][4]) {
#pragma unroll
      for (int n2 = 0; n2 < NT / 2; ++n2) {
        Step<LV == 2, 8> s;
#pragma unroll
        for (int j = NP - 1; j >= 0; --j) {
          uint32_t kb[4], hb[4];
          ldsm4_t(kb, at_bt<ROWB>(st + j * Cfg::kTileK, lane, col0 + n2 * 16, kk));
          if (hb_off != 0)
            ldsm4_t(hb, at_bt<ROWB>(st + hb_off + j * Cfg::kTileK, lane, col0 + n2 * 16, kk));
#pragma unroll
          for (int i = LV - j; i >= 0; --i)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
              uint32_t fh[4], fx[4];
              if (trans) {
                ldsm4_t(fh, at_at<MROW>(st + hs + i * Cfg::kMat, lane, wr * 32 + m * 16, kk));
                ldsm4_t(fx, at_at<MROW>(st + xs + i * Cfg::kMat, lane, wr * 32 + m * 16, kk));
              } else {
                ldsm4(fh, at_a<MROW>(st + hs + i * Cfg::kMat, lane, wr * 32 + m * 16, kk));
                ldsm4(fx, at_a<MROW>(st + xs + i * Cfg::kMat, lane, wr * 32 + m * 16, kk));
              }
              const uint32_t(&b)[4] = hb_off != 0 ? hb : kb;
              s.mma(4 * m, h_acc[m][2 * n2], fh, b[0], b[1]);
              s.mma(4 * m + 1, h_acc[m][2 * n2 + 1], fh, b[2], b[3]);
              s.mma(4 * m + 2, x_acc[m][2 * n2], fx, kb[0], kb[1]);
              s.mma(4 * m + 3, x_acc[m][2 * n2 + 1], fx, kb[2], kb[3]);
            }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          s.add(4 * m, h_acc[m][2 * n2]);
          s.add(4 * m + 1, h_acc[m][2 * n2 + 1]);
          s.add(4 * m + 2, x_acc[m][2 * n2]);
          s.add(4 * m + 3, x_acc[m][2 * n2 + 1]);
        }
      }
    };
    if (left) product(Cfg::oHb, Cfg::oXb, false, 0, aq, ar);
    if (right) product(Cfg::oHs, Cfg::oXd, true, Cfg::oQ, aw, aw);
  }

#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int i = wr * 32 + m * 16 + r * 8 + g4;
      const float be = beta[i];
      float reads = 0.f, writes = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int col = col0 + n * 8 + 2 * t4;
        const float2 kv = kq_pair(0, i, col), qv = kq_pair(Cfg::oQ, i, col);
        const float q0 = aq[m][n][2 * r], q1 = aq[m][n][2 * r + 1];
        const float r0 = ar[m][n][2 * r], r1 = ar[m][n][2 * r + 1];
        const float w0 = aw[m][n][2 * r], w1 = aw[m][n][2 * r + 1];
        reads = fmaf(qv.x, q0, fmaf(qv.y, q1, fmaf(kv.x, r0, fmaf(kv.y, r1, reads))));
        writes = fmaf(kv.x, w0, fmaf(kv.y, w1, writes));
        const float k0 = fmaf(be, w0, r0), k1 = fmaf(be, w1, r1);
        if (i < rows && col < p.dk) {
          if (p.dq_part != nullptr) {
            const int64_t o = ((b * p.L + t0 + i) * p.heads + h) * p.dk + col;
            *reinterpret_cast<float2*>(p.dq_part + o) = make_float2(q0, q1);
            *reinterpret_cast<float2*>(p.dk_part + o) = make_float2(k0, k1);
          } else {
            const int64_t o = kf + (int64_t)i * kstride + col;
            T* dq = static_cast<T*>(p.dq) + o;
            T* dk = static_cast<T*>(p.dk_out) + o;
            if constexpr (sizeof(T) == 4) {
              *reinterpret_cast<float2*>(dq) = make_float2(q0, q1);
              *reinterpret_cast<float2*>(dk) = make_float2(k0, k1);
            } else {
              *reinterpret_cast<uint32_t*>(dq) = pack2<T>(q0, q1);
              *reinterpret_cast<uint32_t*>(dk) = pack2<T>(k0, k1);
            }
          }
        }
      }
      put_row(0, i, reads);
      put_row(1, i, writes);
    }
  __syncthreads();

  // dbeta, and the suffix sums of dlog_decay: one warp, two tokens a lane, in 64 bits
  if (warp == 0) {
    double dg[2], state = 0.0;
    float db[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = 2 * lane + c;
      auto sum4 = [&](int which) {
        return (s_red[which][0][i] + s_red[which][1][i]) + (s_red[which][2][i] + s_red[which][3][i]);
      };
      db[c] = sum4(1);
      dg[c] = (double)sum4(0) - (double)beta[i] * (double)db[c];
      state += (double)beta[i] * (double)sum4(2);
    }
#pragma unroll
    for (int w = 0; w < NTH / 32; ++w)
      if (lane == 0) state += (double)enter[kChunk - 1] * (double)s_dot[w];
    double suffix = dg[0] + dg[1];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double o = __shfl_down_sync(0xffffffffu, suffix, d);
      if (lane + d < 32) suffix += o;
      state += __shfl_xor_sync(0xffffffffu, state, d);
    }
    const double out[2] = {suffix + state, suffix - dg[0] + state};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int i = 2 * lane + c;
      if (i < rows) {
        const int64_t o = (b * p.L + t0 + i) * p.heads + h;
        // a decay of exactly 0 has no slope in its logarithm
        const bool reset = Elem<T>::load(static_cast<const T*>(p.log_decay)[o]) < kDecayFloor;
        static_cast<T*>(p.dlog_decay)[o] = Elem<T>::store(reset ? 0.f : (float)out[c]);
        static_cast<T*>(p.dbeta)[o] = Elem<T>::store(db[c]);
      }
    }
  }
}

// ------------------------------------------------------------------ shared key heads
struct GroupParams {
  const float* src[2];   // (tokens, heads, dk)
  void* dst[2];          // (tokens, key_heads, dk)
  int64_t n;             // tokens x key_heads x dk / 4
  int group, dk4;
};

template <typename T>
__global__ void __launch_bounds__(256) delta_group_kernel(const GroupParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int which = blockIdx.x & 1;
  const int64_t step = (int64_t)(gridDim.x / 2) * blockDim.x;
  for (int64_t i = (int64_t)(blockIdx.x / 2) * blockDim.x + threadIdx.x; i < p.n; i += step) {
    const int64_t head = i / p.dk4;
    const int c = (int)(i - head * p.dk4);
    const float4* src = reinterpret_cast<const float4*>(p.src[which]) + head * p.group * p.dk4 + c;
    float4 s = src[0];
    for (int q = 1; q < p.group; ++q) {
      const float4 x = src[(int64_t)q * p.dk4];
      s.x += x.x;
      s.y += x.y;
      s.z += x.z;
      s.w += x.w;
    }
    T* dst = static_cast<T*>(p.dst[which]) + i * 4;
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<float4*>(dst) = s;
    else
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
  }
}

// ------------------------------------------------------------------ host side
template <typename T, int LV, int DKP, int NW>
cudaError_t rev_nw(const DeltaArgs& a, RevParams& p, int64_t bh) {
  using Cfg = RevCfg<kParts<T>, LV, DKP, NW>;
  auto kern = delta_rev_kernel<T, kParts<T>, LV, DKP, NW>;
  const cudaError_t e =
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return e;
  p.slices = (int)((a.dv + NW * 16 - 1) / (NW * 16));
  return launch_pdl(kern, (unsigned)(bh * p.slices), NW * 32, Cfg::kSmem, a.stream, p);
}

template <typename T, int LV, int DKP>
cudaError_t bwd_pass(const DeltaArgs& a, const DeltaPlan& pl, int64_t b0, int64_t nb) {
  constexpr int NP = kParts<T>;
  cudaError_t e = delta_fwd_pass<T, LV, DKP>(a, pl, b0, nb, true);
  if (e != cudaSuccess) return e;
  char* ws = static_cast<char*>(a.workspace);
  auto bf = [&](int64_t off) { return reinterpret_cast<__nv_bfloat16*>(ws + off); };
  const int64_t k0 = b0 * a.seqlen * a.key_heads * a.dk, v0 = b0 * a.seqlen * a.heads * a.dv;
  const int64_t g0 = b0 * a.seqlen * a.heads, s0 = b0 * a.heads * a.dv * a.dk;
  const int64_t tok = nb * a.seqlen, bh = nb * a.heads;

  RevParams r{};
  if (NP > 1) {
    r.q = bf(pl.q_parts);
    r.k = bf(pl.k_parts);
    r.grad = bf(pl.do_parts);
    r.part_stride = tok * a.key_heads * a.dk;
    r.grad_stride = tok * a.heads * a.dv;
  } else {
    r.q = static_cast<const __nv_bfloat16*>(a.q) + k0;
    r.k = static_cast<const __nv_bfloat16*>(a.k) + k0;
    r.grad = static_cast<const __nv_bfloat16*>(a.grad_out) + v0;
  }
  r.n_mat = bf(pl.n_mat);
  r.p_mat = bf(pl.p_mat);
  r.vecs = reinterpret_cast<const float*>(ws + pl.vecs);
  r.grad_final = a.grad_final ? a.grad_final + s0 : nullptr;
  r.dinitial = a.dinitial ? a.dinitial + s0 : nullptr;
  r.dv_out = static_cast<T*>(a.dv_out) + v0;
  r.dv_parts = bf(pl.dv_parts);
  r.ds_parts = bf(pl.ds_parts);
  r.L = a.seqlen;
  r.chunks = pl.chunks;
  r.key_heads = (int)a.key_heads;
  r.heads = (int)a.heads;
  r.dk = (int)a.dk;
  r.dv = (int)a.dv;
  r.scale = a.scale;
  const bool narrow = bh * ((a.dv + 127) / 128) < a.num_sms || a.dv <= 64;
  e = narrow ? rev_nw<T, LV, DKP, 4>(a, r, bh) : rev_nw<T, LV, DKP, 8>(a, r, bh);
  if (e != cudaSuccess) return e;

  GradParams g{};
  g.q = r.q;
  g.k = r.k;
  g.grad = r.grad;
  g.part_stride = r.part_stride;
  g.grad_stride = r.grad_stride;
  g.e_parts = bf(pl.e_parts);
  g.dv_parts = r.dv_parts;
  g.s_parts = bf(pl.s_parts);
  g.ds_parts = r.ds_parts;
  g.vecs = r.vecs;
  g.log_decay = static_cast<const T*>(a.log_decay) + g0;
  T* dq = static_cast<T*>(a.dq) + k0;
  T* dk = static_cast<T*>(a.dk_out) + k0;
  const bool shared = a.heads != a.key_heads;
  g.dq = dq;
  g.dk_out = dk;
  g.dq_part = shared ? reinterpret_cast<float*>(ws + pl.dq_part) : nullptr;
  g.dk_part = shared ? reinterpret_cast<float*>(ws + pl.dk_part) : nullptr;
  g.dlog_decay = static_cast<T*>(a.dlog_decay) + g0;
  g.dbeta = static_cast<T*>(a.dbeta) + g0;
  g.L = a.seqlen;
  g.chunks = pl.chunks;
  g.key_heads = (int)a.key_heads;
  g.heads = (int)a.heads;
  g.dk = (int)a.dk;
  g.dv = (int)a.dv;
  g.scale = a.scale;
  using GC = GradCfg<NP, LV, DKP>;
  auto kern = delta_grad_kernel<T, NP, LV, DKP>;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GC::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_pdl(kern, (unsigned)(bh * pl.chunks), kGradThreads, GC::kSmem, a.stream, g);
  if (e != cudaSuccess || !shared) return e;

  GroupParams s{};
  s.src[0] = g.dq_part;
  s.src[1] = g.dk_part;
  s.dst[0] = dq;
  s.dst[1] = dk;
  s.n = tok * a.key_heads * (a.dk / 4);
  s.group = (int)(a.heads / a.key_heads);
  s.dk4 = (int)(a.dk / 4);
  const unsigned grid = 2 * (unsigned)std::min<int64_t>((s.n + 255) / 256, 8 * a.num_sms);
  return launch_pdl(delta_group_kernel<T>, grid, 256, 0, a.stream, s);
}

template <typename T, int LV>
cudaError_t bwd_all(const DeltaArgs& a, const DeltaPlan& pl) {
  for (int64_t b0 = 0; b0 < a.batch; b0 += pl.batch) {
    const int64_t nb = std::min(pl.batch, a.batch - b0);
    const cudaError_t e = pl.dkp == 64 ? bwd_pass<T, LV, 64>(a, pl, b0, nb)
                                       : bwd_pass<T, LV, 128>(a, pl, b0, nb);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t launch_delta_bwd(const DeltaArgs& a) {
  const DeltaPlan pl = delta_plan(a.batch, a.seqlen, a.key_heads, a.heads, a.dk, a.dv, a.dtype,
                                  a.wide != 0, true);
  switch (a.dtype) {
    case kF32:
      return bwd_all<float, 2>(a, pl);
    case kF16:
      return a.wide ? bwd_all<__half, 2>(a, pl) : bwd_all<__half, 1>(a, pl);
    default:
      return a.wide ? bwd_all<__nv_bfloat16, 2>(a, pl) : bwd_all<__nv_bfloat16, 1>(a, pl);
  }
}

}  // namespace fpscan
