// Differential attention, backward: dK and dV (the mathematics and the row
// numbering are in diff_attn.h). With c_0 = 1, c_1 = -lam and the saved row
// sums, P_m = 2^(scale log2 e S_m - lse_m),
//
//   dP = dO V^T            (both maps share it: their outputs differ by c_m only)
//   dS_m = c_m P_m (dP - delta_m)
//   dV = sum over rows of (P_0 - lam P_1)^T dO,   dK_m = scale sum over rows of dS_m^T Q_m.
//
// One workgroup = 4 waves = 128 keys of one (b, key head), 32 keys a wave; the
// tokens that see them come through LDS in tiles of 32, one query head of the
// group after the other, so that nothing is added up across workgroups and the
// result does not depend on their order. Scores are formed with tokens in the
// registers and keys over the lanes, so that P and dS turn into the A operands
// of dV and dK where they stand; Q and dO come back as B operands through the
// transposing LDS read.
#include "diff_attn.h"

namespace tj {
namespace {

// WHAT: 1 dV, 2 dK, 3 both. Heads past 64 dims do not have the registers for
// both and form the scores twice.
template <typename T, int HD, int WHAT>
__global__ __launch_bounds__(kDiffThreads, (sizeof(T) == 2 && (HD <= 64 || WHAT == 1) ? 2 : 1)) void diff_bwd_kv_kernel(DiffArgs a) {
  constexpr int DVP = 2 * HD, KS = HD / 16, VS = DVP / 16, KB = HD / 32, VB = DVP / 32, BM = 32;
  constexpr bool DO_DV = (WHAT & 1) != 0, DO_DK = (WHAT & 2) != 0;
  using QT = LdsRows<T, HD>;
  using OT = LdsRows<T, DVP>;
  constexpr int kTile = BM * (2 * HD + DVP);  // Q's two heads and dO
  // V's rows of the workgroup's keys stay in LDS where their fragments would
  // take a wave's registers past what two waves per SIMD have.
  constexpr bool kVInLds = DO_DK && sizeof(T) == 2 && HD == 64;
  __shared__ __attribute__((aligned(1024))) T smem[2][kTile];
  __shared__ __attribute__((aligned(1024))) T sv[kVInLds ? 128 * DVP : 8];
  // lse_0, lse_1 (with the lift), -delta_0 and lam delta_1 (lifted) of a tile's tokens
  __shared__ __attribute__((aligned(16))) float stat[2][4][BM];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, hl = lane / 32,
            ln = lane % 32;
  const DiffTile t = diff_tile(a, blockIdx.x, a.n_mtiles);
  const int L = diff_len(a, t.b);
  const int k0 = t.tile * 128, kw0 = k0 + 32 * w, key = kw0 + ln;
  const bool live = key < L;

  const T* qp = reinterpret_cast<const T*>(a.q) + a.vq.row(t.b, 2 * t.hk * a.G, 0);
  const T* op = reinterpret_cast<const T*>(a.dout) + a.vdo.row(t.b, t.hk * a.G, 0);
  KeyCopy<T, HD, BM, 4> qcopy;
  KeyCopy<T, DVP, BM, 4> ocopy;
  qcopy.init(a.vq.ss, a.D, w, lane);
  ocopy.init(a.vdo.ss, a.Dv, w, lane);
  // Tiles of the group's heads: head g of it, tokens i0 .. i0 + 31.
  auto issue = [&](int g, int i0, T* tile) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      qcopy.issue(qp + (2 * g + c) * a.vq.sh + i0 * a.vq.ss, a.vq.ss, L - i0, a.D, tile + c * BM * HD, w);
    ocopy.issue(op + g * a.vdo.sh + i0 * a.vdo.ss, a.vdo.ss, L - i0, a.Dv, tile + 2 * BM * HD, w);
  };
  // Thread tid < 128 carries number tid / 32 of token tid % 32.
  const float* sp = tid < 64 ? a.lse : a.delta;
  auto load_stat = [&](int g, int i0) {
    const int i = i0 + tid % BM;
    return tid < 128 && i < L ? sp[map_at(a, t.b, t.hk * a.G + g, (tid / BM) & 1, i)] : 0.f;
  };

  frag_t<T> kf[2][KS], vf[DO_DK && !kVInLds ? VS : 1];
  {
    const T* kp = reinterpret_cast<const T*>(a.k) + a.vk.row(t.b, 2 * t.hk, live ? key : 0);
    const T* vp = reinterpret_cast<const T*>(a.v) + a.vv.row(t.b, t.hk, live ? key : 0);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[c][s] = load_frag<T>(live ? kp + c * a.vk.sh : nullptr, 16 * s + 8 * hl, a.D);
    if constexpr (kVInLds) {
      KeyCopy<T, DVP, 128, 4> vcopy;
      vcopy.init(a.vv.ss, a.Dv, w, lane);
      vcopy.issue(reinterpret_cast<const T*>(a.v) + a.vv.row(t.b, t.hk, k0), a.vv.ss, L - k0, a.Dv, sv, w);
    } else if constexpr (DO_DK)
#pragma unroll
      for (int s = 0; s < VS; ++s) vf[s] = load_frag<T>(live ? vp : nullptr, 16 * s + 8 * hl, a.Dv);
  }
  float16_t dv[DO_DV ? VB : 1], dk[2][DO_DK ? KB : 1];
#pragma unroll
  for (auto& x : dv) x = zero16();
#pragma unroll
  for (auto& x : dk[0]) x = zero16();
#pragma unroll
  for (auto& x : dk[1]) x = zero16();

  float lam_max = 0.f;
  for (int g = 0; g < a.G; ++g) {
    const float l = fabsf(a.lam[(t.hk * a.G + g) * a.lam_step]);
    if (l < 3e38f) lam_max = fmaxf(lam_max, l);
  }
  // P is lifted by pl in its exponent; what multiplies P to dS takes that out again.
  const float pl = p_lift<T>(lam_max), dl = ds_lift<T>(a, t.bh, t.hk, lane), log_pl = log2f(pl);
  const float lift = dl / pl;
  const float c2 = a.scale * kLog2e;
  const int i_begin = a.causal ? k0 : 0;
  if (i_begin < L) {
    issue(0, i_begin, smem[0]);
    float next = load_stat(0, i_begin);
    int cur = 0;
    for (int g = 0, i0 = i_begin; g < a.G; cur ^= 1) {
      const float lam = a.lam[(t.hk * a.G + g) * a.lam_step];
      wait_copies();
      if (tid < 128) {
        const int n = tid / BM;
        // A token that is not there weighs nothing: P = 2^(0 - inf).
        const bool in = i0 + tid % BM < L;
        stat[cur][n][tid % BM] = n < 2 ? (in ? next - log_pl : __builtin_inff()) : next * (n == 2 ? -lift : lam * lift);
      }
      wait_lds();
      lds_barrier();
      int g1 = g, i1 = i0 + BM;
      if (i1 >= L) {
        i1 = i_begin;
        ++g1;
      }
      if (g1 < a.G) {
        issue(g1, i1, smem[cur ^ 1]);
        next = load_stat(g1, i1);
      }
      const T *sq[2] = {smem[cur], smem[cur] + BM * HD}, *so = smem[cur] + 2 * BM * HD;
      if (!a.causal || i0 + BM > kw0) {  // else every token stands before the wave's keys
        float16_t p[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          p[c] = zero16();
#pragma unroll
          for (int s = 0; s < KS; ++s) p[c] = Elem<T>::mma(QT::row_frag(sq[c], ln, 16 * s + 8 * hl), kf[c][s], p[c]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4_t ls = *reinterpret_cast<const float4_t*>(&stat[cur][c][8 * q + 4 * hl]);
#pragma unroll
            for (int j = 0; j < 4; ++j) p[c][4 * q + j] = fast_exp2(fmaf(p[c][4 * q + j], c2, -ls[j]));
          }
          if (a.causal && i0 < kw0 + 31) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (i0 + acc_row(r, hl) < key) p[c][r] = 0.f;
          }
        }
        if constexpr (DO_DV) {
          float16_t mix;
#pragma unroll
          for (int r = 0; r < 16; ++r) mix[r] = fmaf(-lam, p[1][r], p[0][r]);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const frag_t<T> f = acc_frag<T>(mix, s);
#pragma unroll
            for (int d = 0; d < VB; ++d) dv[d] = Elem<T>::mma(f, OT::col_frag(so, 16 * s, 32 * d, lane), dv[d]);
          }
        }
        if constexpr (DO_DK) {
          float16_t dp = zero16();
#pragma unroll
          for (int s = 0; s < VS; ++s) {
            const frag_t<T> v = kVInLds ? OT::row_frag(sv, 32 * w + ln, 16 * s + 8 * hl) : vf[kVInLds ? 0 : s];
            dp = Elem<T>::mma(OT::row_frag(so, ln, 16 * s + 8 * hl), v, dp);
          }
          const float nl = -lam * lift;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4_t d0 = *reinterpret_cast<const float4_t*>(&stat[cur][2][8 * q + 4 * hl]);
            const float4_t d1 = *reinterpret_cast<const float4_t*>(&stat[cur][3][8 * q + 4 * hl]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = dp[4 * q + j];
              p[0][4 * q + j] *= fmaf(x, lift, d0[j]);
              p[1][4 * q + j] *= fmaf(x, nl, d1[j]);
            }
          }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const frag_t<T> f = acc_frag<T>(p[c], s);
#pragma unroll
              for (int d = 0; d < KB; ++d) dk[c][d] = Elem<T>::mma(f, QT::col_frag(sq[c], 16 * s, 32 * d, lane), dk[c][d]);
            }
        }
      }
      g = g1;
      i0 = i1;
    }
  }

  // Keys at or past the length have no gradient: zeros, whatever their scores were.
  const float dv_scale = 1.f / pl, dk_scale = a.scale / dl;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = kw0 + acc_row(r, hl);
    if (j >= a.Sk) continue;
    const bool in = j < L;
    if constexpr (DO_DV) {
      T* p = reinterpret_cast<T*>(a.dv) + a.vdv.row(t.b, t.hk, j);
#pragma unroll
      for (int d = 0; d < VB; ++d)
        if (32 * d + ln < a.Dv) p[32 * d + ln] = (T)(in ? dv[d][r] * dv_scale : 0.f);
    }
    if constexpr (DO_DK) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        T* p = reinterpret_cast<T*>(a.dk) + a.vdk.row(t.b, 2 * t.hk + c, j);
#pragma unroll
        for (int d = 0; d < KB; ++d)
          if (32 * d + ln < a.D) p[32 * d + ln] = (T)(in ? dk[c][d][r] * dk_scale : 0.f);
      }
    }
  }
}

template <typename T, int HD, int WHAT>
int launch(const DiffArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((diff_bwd_kv_kernel<T, HD, WHAT>), dim3(uint32_t((int64_t)a.B * a.Hk * a.n_mtiles)),
                     dim3(kDiffThreads), 0, stream, a);
  return tjh::launch_status();
}

}  // namespace

int diff_bwd_kv(const DiffArgs& args, int dtype, hipStream_t stream) {
  return diff_dispatch(args, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    DiffArgs a = args;
    a.n_mtiles = (a.Sk + 127) / 128;
    if constexpr (HD == 128) {
      const int rc = launch<T, HD, 1>(a, stream);
      return rc != TJ_OK ? rc : launch<T, HD, 2>(a, stream);
    } else {
      return launch<T, HD, 3>(a, stream);
    }
  });
}

}  // namespace tj
