// Differential attention, backward: dK and dV (the mathematics and the row
// numbering are in diff_attn.h). With c_0 = 1, c_1 = -lam and the saved row
// sums, P_m = 2^(scale log2 e S_m - lse_m),
//
//   dP = dO V^T            (both maps share it: their outputs differ by c_m only)
//   dS_m = c_m P_m (dP - delta_m)
//   dV = sum over rows of (P_0 - lam P_1)^T dO,   dK_m = scale sum over rows of dS_m^T Q_m.
//
// One workgroup = KB blocks of 32 keys of one (b, key head) times RG
// groups of token tiles, a wave each: the tiles of 32 tokens that see the keys, of one query
// head of the group after the other, are dealt to the groups in turn, and the
// groups' sums meet in LDS at the end. So nothing is added up across
// workgroups, the result does not depend on their order, and a causal launch
// has many workgroups of unequal length to fill the chip with, longest first.
// Scores are formed with tokens in the registers and keys over the lanes, so
// that P and dS turn into the A operands of dV and dK where they stand; Q and dO
// come back as B operands through the transposing LDS read. 16-bit inputs have the
// mixed P and dS rounded to their type for these products, one rounding more than
// the result's own (fp32 MFMAs would take 16 times as long); fp32 inputs have none.
//
// b2 h8 key heads 4 s4096 d64 bf16 causal: 209 us, 657 TFLOP/s of its 8D + 4Dv
// operations a pair; matrix units busy 34 % of the time, vector units 42 %, LDS 31 %
// without bank conflicts: a step's phases depend on each other, and the two
// waves of a SIMD meet in the same ones. LDS reads issued further ahead, and the
// rows' numbers out of the way of the copies, gained 2 % together.
#include "diff_attn.h"

namespace tj {
namespace {

// WHAT: 1 dV, 2 dK, 3 both; fp32 heads past 64 dims do not have the registers for
// both and form the scores twice. (16-bit ones of 128 dims do, in all 512 registers
// of one wave a SIMD with operands read ahead: 229 us instead of 228 + 217 at b2 h4
// s4096 bf16.) Eight waves, two a SIMD, where their registers allow it, else four;
// as many groups as have room for two tiles each (at most 128 KB of LDS), so that a
// tile is on its way while one is worked on.
// HALF: half of the key blocks, and so of the waves, a workgroup.
template <typename T, int HD, int WHAT, bool HALF>
struct KvShape {
  static constexpr int DVP = 2 * HD;
  static constexpr int kWhole = (sizeof(T) == 2 && HD <= 64) || HD == 32 ? 8 : 4, WAVES = HALF ? kWhole / 2 : kWhole;
  static constexpr int RG = 512 / (HD * (int)sizeof(T)) < kWhole / 2 ? 512 / (HD * (int)sizeof(T)) : kWhole / 2;
  static constexpr int KB = WAVES / RG;
  // What of the keys' rows stays in LDS, as the registers have no room for it.
  static constexpr bool kK1InLds = WHAT == 3 && HD == 128;
  static constexpr bool kVInLds = (WHAT & 2) != 0 && sizeof(T) == 2 && HD == 64;
  // bf16, two deep: 354 -> 337 us (fp32 d64, one deep), 214 -> 209 (bf16 d64), none at d32 (319).
  static constexpr int kDepth = HD == 32 ? 0 : sizeof(T) == 2 ? 2 : 1;
  static constexpr int kTile = 32 * (2 * HD + DVP);  // Q's two heads and dO, of 32 tokens
  static constexpr int kBytes = kTile * (int)sizeof(T), kHead = 32 * HD * (int)sizeof(T);
};

template <typename T, int HD, int WHAT, bool HALF>
__global__ __launch_bounds__((64 * KvShape<T, HD, WHAT, HALF>::WAVES), (KvShape<T, HD, WHAT, HALF>::WAVES / 4)) void diff_bwd_kv_kernel(DiffArgs a) {
  using SH = KvShape<T, HD, WHAT, HALF>;
  constexpr int DVP = SH::DVP, KS = HD / 16, VS = DVP / 16, DB = HD / 32, VB = DVP / 32, BM = 32;
  constexpr int KB = SH::KB, RG = SH::RG, WAVES = SH::WAVES;
  constexpr bool DO_DV = (WHAT & 1) != 0, DO_DK = (WHAT & 2) != 0;
  using QT = LdsRows<T, HD>;
  using OT = LdsRows<T, DVP>;
  __shared__ __attribute__((aligned(1024))) T smem[RG][2][SH::kTile];
  __shared__ __attribute__((aligned(1024))) T sv[SH::kVInLds ? 32 * KB * DVP : 8];
  __shared__ __attribute__((aligned(1024))) T sk[SH::kK1InLds ? 32 * KB * HD : 8];
  __shared__ __attribute__((aligned(1024))) float stat[RG][2][4][BM];  // of a tile's tokens
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, hl = lane / 32,
            ln = lane % 32;
  const int kb = w % KB, rg = w / KB;
  const DiffTile t = diff_tile(a, blockIdx.x, a.n_mtiles);
  const int L = diff_len(a, t.b);
  const int k0 = t.tile * 32 * KB, kw0 = k0 + 32 * kb, key = kw0 + ln;
  const bool live = key < L;

  // The group's KB waves bring its tiles.
  const T* qp = reinterpret_cast<const T*>(a.q) + a.vq.row(t.b, 2 * t.hk * a.G, 0);
  const T* op = reinterpret_cast<const T*>(a.dout) + a.vdo.row(t.b, t.hk * a.G, 0);
  KeyCopy<T, HD, BM, KB> qcopy;
  KeyCopy<T, DVP, BM, KB> ocopy;
  qcopy.init(a.vq.ss, a.D, kb, lane);
  ocopy.init(a.vdo.ss, a.Dv, kb, lane);
  const uint32_t group = lds_offset(smem[rg]);
  const uint32_t qrow = QT::lane_row(lane), qcol = QT::lane_col(lane), orow = OT::lane_row(lane) + 2 * SH::kHead,
                 ocol = OT::lane_col(lane) + 2 * SH::kHead;
  const uint32_t krow = lds_offset(sk) + QT::lane_row(lane) + 32 * kb * QT::kRowBytes;
  const uint32_t vrow = lds_offset(sv) + OT::lane_row(lane) + 32 * kb * OT::kRowBytes;
  // Tile n: head n / tiles of the group, tokens i_begin + 32 (n % tiles) on.
  const int i_begin = a.causal ? k0 : 0;
  const int tiles = k0 < L ? (L - i_begin + BM - 1) / BM : 0, n_end = tiles * a.G;
  // `n` tiles further on: the head and the token (no division in the loop).
  auto advance = [&](int& g, int& i0, int n) {
    i0 += BM * n;
    while (i0 >= i_begin + BM * tiles) {
      i0 -= BM * tiles;
      ++g;
    }
  };
  auto issue = [&](int g, int i0, uint32_t tile) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      qcopy.issue(qp + (2 * g + c) * a.vq.sh + i0 * a.vq.ss, a.vq.ss, L - i0, a.D, tile + c * SH::kHead, kb);
    ocopy.issue(op + g * a.vdo.sh + i0 * a.vdo.ss, a.vdo.ss, L - i0, a.Dv, tile + 2 * SH::kHead, kb);
  };
  // The tokens' numbers by the same way (a load into registers would have to be
  // waited for, and every copy issued before with it), two rows of 32 an instruction.
  const uint32_t stat0 = lds_offset(stat[rg]);
  auto issue_stat = [&](int g, int i0, int buf) {
#pragma unroll
    for (int pair = 0; pair < 2; ++pair)
      if (kb == pair % KB)
        copy_4(make_rsrc(stat_at(a, t.b, t.hk * a.G + g, i0, 2 * pair), 256), stat0 + (buf * 2 + pair) * 256, 4 * lane);
  };

  frag_t<T> kf[SH::kK1InLds ? 1 : 2][KS], vf[DO_DK && !SH::kVInLds ? VS : 1];
  {
    const T* kp = reinterpret_cast<const T*>(a.k) + a.vk.row(t.b, 2 * t.hk, live ? key : 0);
    const T* vp = reinterpret_cast<const T*>(a.v) + a.vv.row(t.b, t.hk, live ? key : 0);
#pragma unroll
    for (int c = 0; c < (SH::kK1InLds ? 1 : 2); ++c)
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[c][s] = load_frag<T>(live ? kp + c * a.vk.sh : nullptr, 16 * s + 8 * hl, a.D);
    if constexpr (SH::kK1InLds) {
      KeyCopy<T, HD, 32 * KB, WAVES> kcopy;
      kcopy.init(a.vk.ss, a.D, w, lane);
      kcopy.issue(reinterpret_cast<const T*>(a.k) + a.vk.row(t.b, 2 * t.hk + 1, k0), a.vk.ss, L - k0, a.D, lds_offset(sk), w);
      wait_copies();
      __syncthreads();
    }
    if constexpr (SH::kVInLds) {
      KeyCopy<T, DVP, 32 * KB, WAVES> vcopy;
      vcopy.init(a.vv.ss, a.Dv, w, lane);
      vcopy.issue(reinterpret_cast<const T*>(a.v) + a.vv.row(t.b, t.hk, k0), a.vv.ss, L - k0, a.Dv, lds_offset(sv), w);
      wait_copies();
      __syncthreads();
    } else if constexpr (DO_DK) {
#pragma unroll
      for (int s = 0; s < VS; ++s) vf[s] = load_frag<T>(live ? vp : nullptr, 16 * s + 8 * hl, a.Dv);
    }
  }
  float16_t dv[DO_DV ? VB : 1], dk[2][DO_DK ? DB : 1];
#pragma unroll
  for (auto& x : dv) x = zero16();
#pragma unroll
  for (auto& x : dk[0]) x = zero16();
#pragma unroll
  for (auto& x : dk[1]) x = zero16();

  const float pl = p_lift<T>(a, t.hk), dl = DsLift<T>(a, t.bh, t.hk, lane).all(), lift = dl / pl;
  const float c2 = a.scale * kLog2e;
  const auto lams = (const __attribute__((address_space(4))) float*)a.lam;
  int g = 0, i0 = i_begin;  // this round's tile
  if (rg < n_end) {
    advance(g, i0, rg);
    issue(g, i0, group);
    issue_stat(g, i0, 0);
  }
  // The workgroup goes round together, the last round maybe without a tile for every group.
  const int rounds = (n_end + RG - 1) / RG;
  for (int round = 0, n = rg, cur = 0; round < rounds; ++round, n += RG, cur ^= 1) {
    const bool on = n < n_end;
    // A scalar load (nothing here writes lam): it does not wait for the copies.
    const float lam = on ? lams[(t.hk * a.G + g) * a.lam_step] : 0.f;
    // The tile is there, and the group's other one has been read by its waves.
    wait_copies();
    lds_barrier();
    const uint32_t tile = group + cur * SH::kBytes, srow = stat0 + cur * 512 + 16 * hl;
    const bool busy = on && (!a.causal || i0 + BM > kw0);  // else every token stands before the wave's keys
    int g1 = g, i1 = i0;
    // Called after the scores: a spilled K fragment, read again for them, would wait for
    // the copies. In both branches rather than between two, where p would be merged.
    auto issue_next = [&] {
      if (n + RG >= n_end) return;
      advance(g1, i1, RG);
      issue(g1, i1, group + (cur ^ 1) * SH::kBytes);
      issue_stat(g1, i1, cur ^ 1);
    };
    if (!busy) issue_next();
    if (busy) {
      float16_t p[2], dp = zero16();
      p[0] = p[1] = zero16();
      struct Two { frag_t<T> o, v; };
      read_ahead<2 * KS, SH::kDepth>(
          [&](int i) {
            const int c = i / KS, s = i % KS;
            return Two{QT::row_frag(tile + qrow, s, c * SH::kHead), SH::kK1InLds && c == 1 ? QT::row_frag(krow, s, 0) : kf[SH::kK1InLds ? 0 : c][s]};
          },
          [&](int i, Two f) { p[i / KS] = Elem<T>::mma(f.o, f.v, p[i / KS]); });
      if constexpr (DO_DK) {
        read_ahead<VS, SH::kDepth>(
            [&](int s) { return Two{OT::row_frag(tile + orow, s, 0), SH::kVInLds ? OT::row_frag(vrow, s, 0) : vf[SH::kVInLds ? 0 : s]}; },
            [&](int, Two f) { dp = Elem<T>::mma(f.o, f.v, dp); });
      }
      issue_next();
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4_t ls = lds_at<float4_t>(srow + c * 128 + q * 32);
#pragma unroll
          for (int j = 0; j < 4; ++j) p[c][4 * q + j] = fast_exp2(fmaf(p[c][4 * q + j], c2, ls[j]));
        }
        if (a.causal && i0 < kw0 + 31) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (i0 + acc_row(r, hl) < key) p[c][r] = 0.f;
        }
      }
      frag_t<T> fm[2], fs[2][2];
      if constexpr (DO_DV) {
        float16_t mix;
#pragma unroll
        for (int r = 0; r < 16; ++r) mix[r] = fmaf(-lam, p[1][r], p[0][r]);
#pragma unroll
        for (int s = 0; s < 2; ++s) fm[s] = acc_frag<T>(mix, s);
      }
      if constexpr (DO_DK) {
        const float nl = -lam * lift;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float4_t d0 = lds_at<float4_t>(srow + 256 + q * 32);
          const float4_t d1 = lds_at<float4_t>(srow + 384 + q * 32);
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
          for (int s = 0; s < 2; ++s) fs[c][s] = acc_frag<T>(p[c], s);
      }
      if constexpr (SH::kDepth > 0) __builtin_amdgcn_sched_barrier(0);
      if constexpr (DO_DV)
        read_ahead<2 * VB, SH::kDepth>([&](int i) { return OT::col_frag(tile + ocol, i % VB, 16 * (i / VB) * OT::kRowBytes); },
                                       [&](int i, frag_t<T> f) { dv[i % VB] = Elem<T>::mma(fm[i / VB], f, dv[i % VB]); });
      if constexpr (DO_DK)
        read_ahead<4 * DB, SH::kDepth>(
            [&](int i) { return QT::col_frag(tile + qcol, i % DB, i / (2 * DB) * SH::kHead + 16 * (i / DB % 2) * QT::kRowBytes); },
            [&](int i, frag_t<T> f) {
              const int c = i / (2 * DB), s = i / DB % 2, d = i % DB;
              dk[c][d] = Elem<T>::mma(fs[c][s], f, dk[c][d]);
            });
    }
    g = g1;
    i0 = i1;
  }

  // The groups' sums, the upper half's added to the lower half's.
  if constexpr (RG > 1) {
    constexpr int NR = (DO_DV ? VB : 0) + (DO_DK ? 2 * DB : 0);
    static_assert(sizeof(smem) >= (RG / 2) * KB * NR * 16 * kWave * sizeof(float), "room for the groups' sums");
    float4_t* x = reinterpret_cast<float4_t*>(smem);
    auto each = [&](auto&& f) {
      int i = 0;
      if constexpr (DO_DV)
#pragma unroll
        for (int d = 0; d < VB; ++d) f(dv[d], i++);
      if constexpr (DO_DK)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int d = 0; d < DB; ++d) f(dk[c][d], i++);
    };
#pragma unroll
    for (int half = RG / 2; half > 0; half /= 2) {
      __syncthreads();
      if (rg >= half && rg < 2 * half)
        each([&](float16_t& v, int i) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            x[((((rg - half) * KB + kb) * NR + i) * 4 + q) * kWave + lane] = float4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        });
      __syncthreads();
      if (rg < half)
        each([&](float16_t& v, int i) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4_t y = x[(((rg * KB + kb) * NR + i) * 4 + q) * kWave + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * q + j] += y[j];
          }
        });
    }
    if (rg != 0) return;
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
        for (int d = 0; d < DB; ++d)
          if (32 * d + ln < a.D) p[32 * d + ln] = (T)(in ? dk[c][d][r] * dk_scale : 0.f);
      }
    }
  }
}

template <typename T, int HD, int WHAT, bool HALF = false>
int launch(DiffArgs a, hipStream_t stream) {
  using SH = KvShape<T, HD, WHAT, HALF>;
  constexpr int kKeys = 32 * SH::KB;
  a.n_mtiles = (a.Sk + kKeys - 1) / kKeys;
  // Where half of the CUs would have no work, us with 64 keys a workgroup / 32: b1 h1 s8192
  // d64 bf16 163 / 138, h2 s4096 87 / 74, h8 s1024 d32 fp32 80 / 53; 192 workgroups of 64: 32 / 36.
  if constexpr (!HALF && SH::WAVES == 8)
    if ((int64_t)a.B * a.Hk * a.n_mtiles <= kCus / 2) return launch<T, HD, WHAT, true>(a, stream);
  hipLaunchKernelGGL((diff_bwd_kv_kernel<T, HD, WHAT, HALF>), dim3(uint32_t((int64_t)a.B * a.Hk * a.n_mtiles)),
                     dim3(64 * SH::WAVES), 0, stream, a);
  return tjh::launch_status();
}

}  // namespace

int diff_bwd_kv(const DiffArgs& args, int dtype, hipStream_t stream) {
  return diff_dispatch(args, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    const DiffArgs& a = args;
    if constexpr (HD == 128 && sizeof(T) == 4) {
      const int rc = launch<T, HD, 1>(a, stream);
      return rc != TJ_OK ? rc : launch<T, HD, 2>(a, stream);
    } else {
      return launch<T, HD, 3>(a, stream);
    }
  });
}

}  // namespace tj
