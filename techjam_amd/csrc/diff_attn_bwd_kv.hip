// Differential attention, backward: dK and dV (the mathematics and the row
// numbering are in diff_attn.h). With c_0 = 1, c_1 = -lam and the saved row
// sums, P_m = 2^(scale log2 e S_m - lse_m),
//
//   dP = dO V^T            (both maps share it: their outputs differ by c_m only)
//   dS_m = c_m P_m (dP - delta_m)
//   dV = sum over rows of (P_0 - lam P_1)^T dO,   dK_m = scale sum over rows of dS_m^T Q_m.
//
// One workgroup = 4 waves = 128 keys of one (b, key head), 32 keys a wave, all
// the rows that see them in turn through LDS; the rows of the G heads that
// share the keys are one list, so nothing is added up across workgroups and the
// result does not depend on their order. Scores are formed with rows in the
// registers and keys over the lanes, so that P and dS turn into the A operands
// of dV and dK where they stand; Q and dO come back as B operands through the
// transposing LDS read.
#include "diff_attn.h"

namespace tj {
namespace {

// WHAT: 1 dV, 2 dK, 3 both. fp32 heads past 64 dims do not have the registers
// for both and form the scores twice.
template <typename T, int HD, int WHAT>
__global__ __launch_bounds__(kDiffThreads, 1) void diff_bwd_kv_kernel(DiffArgs a) {
  constexpr int DVP = 2 * HD, KS = HD / 16, VS = DVP / 16, KB = HD / 32, VB = DVP / 32, BM = 32;
  constexpr bool DO_DV = (WHAT & 1) != 0, DO_DK = (WHAT & 2) != 0;
  using QT = LdsRows<T, HD>;
  using OT = LdsRows<T, DVP>;
  __shared__ __attribute__((aligned(16))) T sq[2][BM * QT::kStride];
  __shared__ __attribute__((aligned(16))) T so[BM * OT::kStride];
  // lse_0, lse_1, delta_0, lam delta_1 (lifted), -lam (lifted), -lam
  __shared__ __attribute__((aligned(16))) float stat[6][BM];
  const int tid = threadIdx.x, w = tid / kWave, lane = tid % kWave, hl = lane / 32, ln = lane % 32;
  const DiffTile t = diff_tile(a, blockIdx.x, a.n_mtiles);
  const int L = diff_len(a, t.b);
  const int k0 = t.tile * 128, kw0 = k0 + 32 * w, key = kw0 + ln;
  const bool live = key < L;

  frag_t<T> kf[2][KS], vf[DO_DK ? VS : 1];
  {
    const T* kp = reinterpret_cast<const T*>(a.k) + a.vk.row(t.b, 2 * t.hk, live ? key : 0);
    const T* vp = reinterpret_cast<const T*>(a.v) + a.vv.row(t.b, t.hk, live ? key : 0);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[c][s] = load_frag<T>(live ? kp + c * a.vk.sh : nullptr, 16 * s + 8 * hl, a.D);
    if constexpr (DO_DK)
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
  const int r_end = k0 < L ? min(a.R, L * a.G) : 0;
  const int r_begin = a.causal ? k0 * a.G / BM * BM : 0;
  const T* qp = reinterpret_cast<const T*>(a.q);
  const T* op = reinterpret_cast<const T*>(a.dout);
  const float* lse = a.lse + (int64_t)t.bh * 2 * a.R;
  const float* del = a.delta + (int64_t)t.bh * 2 * a.R;
  for (int r0 = r_begin; r0 < r_end; r0 += BM) {
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 2; ++c)
      QT::template fill<BM>(sq[c], tid, a.D, [&](int row) {
        const int r = r0 + row;
        return r < r_end ? qp + a.vq.row(t.b, 2 * (t.hk * a.G + r % a.G) + c, r / a.G) : nullptr;
      });
    OT::template fill<BM>(so, tid, a.Dv, [&](int row) {
      const int r = r0 + row;
      return r < r_end ? op + a.vdo.row(t.b, t.hk * a.G + r % a.G, r / a.G) : nullptr;
    });
    if (tid < BM) {
      const int r = r0 + tid;
      const bool in = r < r_end;
      const float lam = a.lam[(t.hk * a.G + (in ? r % a.G : 0)) * a.lam_step];
      // A row that is not there weighs nothing: P = 2^(0 - inf).
      stat[0][tid] = in ? lse[r] - log_pl : __builtin_inff();
      stat[1][tid] = in ? lse[a.R + r] - log_pl : __builtin_inff();
      stat[2][tid] = in ? -del[r] * lift : 0.f;
      stat[3][tid] = in ? lam * del[a.R + r] * lift : 0.f;
      stat[4][tid] = in ? -lam * lift : 0.f;
      stat[5][tid] = in ? -lam : 0.f;
    }
    __syncthreads();
    if (a.causal && min(r0 + BM, r_end) - 1 < kw0 * a.G) continue;  // every row stands before the wave's keys

    float16_t p[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      p[c] = zero16();
#pragma unroll
      for (int s = 0; s < KS; ++s) p[c] = Elem<T>::mma(QT::row_frag(sq[c], ln, 16 * s + 8 * hl), kf[c][s], p[c]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4_t ls = *reinterpret_cast<const float4_t*>(&stat[c][8 * q + 4 * hl]);
#pragma unroll
        for (int j = 0; j < 4; ++j) p[c][4 * q + j] = fast_exp2(fmaf(p[c][4 * q + j], c2, -ls[j]));
      }
      if (a.causal && r0 < (kw0 + 31) * a.G) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (r0 + acc_row(r, hl) < key * a.G) p[c][r] = 0.f;
      }
    }
    if constexpr (DO_DV) {
      float16_t mix;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4_t nl = *reinterpret_cast<const float4_t*>(&stat[5][8 * q + 4 * hl]);
#pragma unroll
        for (int j = 0; j < 4; ++j) mix[4 * q + j] = fmaf(nl[j], p[1][4 * q + j], p[0][4 * q + j]);
      }
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
      for (int s = 0; s < VS; ++s) dp = Elem<T>::mma(OT::row_frag(so, ln, 16 * s + 8 * hl), vf[s], dp);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4_t d0 = *reinterpret_cast<const float4_t*>(&stat[2][8 * q + 4 * hl]);
        const float4_t d1 = *reinterpret_cast<const float4_t*>(&stat[3][8 * q + 4 * hl]);
        const float4_t nl = *reinterpret_cast<const float4_t*>(&stat[4][8 * q + 4 * hl]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = dp[4 * q + j];
          p[0][4 * q + j] *= fmaf(x, lift, d0[j]);
          p[1][4 * q + j] *= fmaf(x, nl[j], d1[j]);
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
    if constexpr (sizeof(T) == 4 && HD == 128) {
      const int rc = launch<T, HD, 1>(a, stream);
      return rc != TJ_OK ? rc : launch<T, HD, 2>(a, stream);
    } else {
      return launch<T, HD, 3>(a, stream);
    }
  });
}

}  // namespace tj
