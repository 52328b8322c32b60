// Differential attention, backward: the rows' sums delta_m = rowsum(dO o O_m)
// beforehand, dQ, and the gradient of the second map's weight (the mathematics
// and the row numbering are in diff_attn.h and diff_attn_bwd_kv.hip).
//
//   dQ_m = scale dS_m K_m,  dS_m = c_m P_m (dP - delta_m)
//   dlam = - sum over rows of sum_j P_1 dP
//
// delta_m comes from the maps' outputs, which the forward pass keeps in fp32:
// rounded to 16 bits they cost dQ and dK a twentieth of their accuracy (bf16,
// causal, 1024 tokens, 64 dims: 2.56e-3 instead of 2.40e-3, relative 2-norm; the
// rounding of dS and of the result is 2.38e-3). What is left of its error is the
// rounding of P in the forward product: the sum of P_m (dP - delta_m) over the
// keys (P_m sums to 1). The dQ kernel adds it back to delta, exact then to what
// fp32 sums are, for dlam and for dK, which come after it, and leaves the rows'
// numbers as the dK, dV kernel wants them. dS itself is rounded to the operands'
// type for the product, as is the result, two roundings where fp32 products
// have one: the error of dQ is 1.45 times theirs at 64 dims and 1.6 at 16, where
// the sum of dS K cancels more (fp32 MFMAs would take 16 times as long).
//
// b2 h8 key heads 4 s4096 d64 bf16 causal: dQ 144 us, 716 TFLOP/s of its 8D + 2Dv
// operations a pair, matrix units busy 39 %, vector units 57 %; delta 14 us, 6 TB/s.
#include "diff_attn.h"

namespace tj {
namespace {

// One group of `lpr` lanes per row: 16-byte chunks of dO and the same columns of the maps' outputs. n_peaks
// blocks share the rows, then the keys, of one (b, key head).
template <typename T>
__global__ __launch_bounds__(kDiffThreads) void diff_delta_kernel(DiffArgs a, int lpr) {
  constexpr int VEC = Vec16<float>::N * (4 / (int)sizeof(T));
  typedef T vec_t __attribute__((ext_vector_type(VEC)));
  __shared__ float red[2][kDiffThreads / kWave];
  const int tid = threadIdx.x, block = blockIdx.x % a.n_peaks, bh = blockIdx.x / a.n_peaks, b = bh / a.Hk, hk = bh % a.Hk;
  const int L = diff_len(a, b);
  const int lane = tid % lpr, per_block = kDiffThreads / lpr;
  const bool on = lane * VEC < a.Dv;
  float peak_o = 0.f, peak_v = 0.f;
  for (int r = block * per_block + tid / lpr; r < a.R; r += a.n_peaks * per_block) {
    const int i = r / a.G, head = hk * a.G + r % a.G;
    float d0 = 0.f, d1 = 0.f, n = 0.f;
    if (i < L && on) {
      const vec_t x = *reinterpret_cast<const vec_t*>(reinterpret_cast<const T*>(a.dout) + a.vdo.row(b, head, i) + lane * VEC);
      const float* mp = a.maps + row_at(a, b, head, i) * 2 * a.Dv + lane * VEC;
#pragma unroll
      for (int e = 0; e < VEC; e += 4) {
        const float4_t y = *reinterpret_cast<const float4_t*>(mp + e), z = *reinterpret_cast<const float4_t*>(mp + a.Dv + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float g = (float)x[e + j];
          d0 = fmaf(g, y[j], d0);
          d1 = fmaf(g, z[j], d1);
          n = fmaf(g, g, n);
        }
      }
    }
    for (int s = lpr / 2; s > 0; s >>= 1) {
      d0 += __shfl_xor(d0, s);
      d1 += __shfl_xor(d1, s);
      n += __shfl_xor(n, s);
    }
    if (lane == 0) {
      a.delta[map_at(a, b, head, 0, i)] = d0;
      a.delta[map_at(a, b, head, 1, i)] = d1;
      if (i == a.Sq - 1)
        for (int j = a.Sq; j < (int)stat_rows(a.Sq); ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) *stat_at(a, b, head, j, c) = c < 2 ? -__builtin_inff() : 0.f;
    }
    if (n < 3e38f) peak_o = fmaxf(peak_o, n);  // not those that are not finite: they spoil their own row only
  }
  if constexpr (std::is_same<T, half_t>::value) {
    for (int j = block * per_block + tid / lpr; j < L; j += a.n_peaks * per_block) {
      float n = 0.f;
      if (on) {
        const vec_t x = *reinterpret_cast<const vec_t*>(reinterpret_cast<const T*>(a.v) + a.vv.row(b, hk, j) + lane * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) n = fmaf((float)x[e], (float)x[e], n);
      }
      for (int s = lpr / 2; s > 0; s >>= 1) n += __shfl_xor(n, s);
      if (n < 3e38f) peak_v = fmaxf(peak_v, n);
    }
    for (int s = kWave / 2; s > 0; s >>= 1) {
      peak_o = fmaxf(peak_o, __shfl_xor(peak_o, s));
      peak_v = fmaxf(peak_v, __shfl_xor(peak_v, s));
    }
    if (tid % kWave == 0) {
      red[0][tid / kWave] = peak_o;
      red[1][tid / kWave] = peak_v;
    }
    __syncthreads();
    if (tid < 2) {
      float x = red[tid][0];
      for (int w = 1; w < kDiffThreads / kWave; ++w) x = fmaxf(x, red[tid][w]);
      a.peak[((int64_t)bh * 2 + tid) * kPeakParts + block] = sqrtf(x);
    }
  }
}

// A workgroup = RB blocks of 32 rows times KG groups, a wave each, keys through
// LDS in tiles of 32 dealt to the groups in turn, whose sums meet in LDS at the
// end. Scores transposed as in the forward kernel: a row's sums are its lane's
// own numbers, and dS turns into the B operand of dQ^T = K^T dS^T. Four waves;
// 128 rows, or 64 with two groups, or 32 with four, if two tiles for each fit.
template <typename T, int HD, int BLOCKS>
struct QShape {
  static constexpr int DVP = 2 * HD;
  static constexpr int WAVES = 4;
  static constexpr int RB = BLOCKS, KG = WAVES / RB;
  static_assert(row_blocks_fit<T, HD>(BLOCKS), "two tiles a group");
  static constexpr int kDepth = HD == 32 ? 0 : 2;  // fp32 d64: 281 -> 271 us (b2 h8 s2048); 16 bits: equal
  static constexpr int kBytes = 32 * (2 * HD + DVP) * (int)sizeof(T), kHead = 32 * HD * (int)sizeof(T);
};

template <typename T, int HD, int BLOCKS>
__global__ __launch_bounds__((64 * QShape<T, HD, BLOCKS>::WAVES), (HD == 32 || (sizeof(T) == 2 && HD == 64) ? 2 : 1)) void
diff_bwd_q_kernel(DiffArgs a) {
  using SH = QShape<T, HD, BLOCKS>;
  constexpr int DVP = SH::DVP, KS = HD / 16, VS = DVP / 16, DB = HD / 32, BN = 32, RB = SH::RB, KG = SH::KG, ROWS = 32 * RB;
  constexpr int kBytes = SH::kBytes, kHead = SH::kHead;
  using KT = LdsRows<T, HD>;
  using VT = LdsRows<T, DVP>;
  constexpr int kSums = KG > 1 ? KG / 2 * RB * (2 * DB * 16 + 2) * kWave * 4 : 0;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[KG * 2 * kBytes > kSums ? KG * 2 * kBytes : kSums];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, hl = lane / 32,
            ln = lane % 32;
  const int kg = w / RB, rb = w % RB;
  const DiffTile t = diff_tile(a, blockIdx.x, a.n_mtiles);
  const int mt = a.n_mtiles - 1 - t.tile;
  const int L = diff_len(a, t.b);
  const int r0 = mt * ROWS, rw0 = r0 + 32 * rb, r = rw0 + ln;
  const int i = r / a.G, head = t.hk * a.G + r % a.G;
  const bool live = r < a.R && i < L;
  const int limit = a.causal ? i : L - 1;
  const int kv_end = r0 / a.G >= L ? 0 : (a.causal ? min(L, min(r0 + ROWS - 1, a.R - 1) / a.G + 1) : L);
  const int own_end = rw0 >= a.R || rw0 / a.G >= L ? 0 : (a.causal ? min(L, min(rw0 + 31, a.R - 1) / a.G + 1) : L);
  const int free = a.causal ? rw0 / a.G : L - 1;

  const T* kp = reinterpret_cast<const T*>(a.k) + a.vk.row(t.b, 2 * t.hk, 0);
  const T* vp = reinterpret_cast<const T*>(a.v) + a.vv.row(t.b, t.hk, 0);
  KeyCopy<T, HD, BN, RB> kcopy;
  KeyCopy<T, DVP, BN, RB> vcopy;
  kcopy.init(a.vk.ss, a.D, rb, lane);
  vcopy.init(a.vv.ss, a.Dv, rb, lane);
  const uint32_t tiles = lds_offset(smem) + kg * 2 * kBytes;
  const uint32_t krow = KT::lane_row(lane), kcol = KT::lane_col(lane), vrow = VT::lane_row(lane) + 2 * kHead;
  auto issue = [&](int kv0, uint32_t tile) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      kcopy.issue(kp + c * a.vk.sh + kv0 * a.vk.ss, a.vk.ss, L - kv0, a.D, tile + c * kHead, rb);
    vcopy.issue(vp + kv0 * a.vv.ss, a.vv.ss, L - kv0, a.Dv, tile + 2 * kHead, rb);
  };
  int kv0 = BN * kg;
  if (kv0 < kv_end) issue(kv0, tiles);

  // Every other token works with -dO and -dP: the matrix unit's sums lean to minus
  // infinity, which dlam, the sum of all rows, would keep (b8 h4 s1024 d64 fp16: its
  // error 3.0e-5 in every one of eight draws, now 0 to 7e-6 of either sign).
  const bool odd = i % 2 != 0;
  const float sign = odd ? -1.f : 1.f;
  frag_t<T> qf[2][KS], of[VS];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + (live ? a.vq.row(t.b, 2 * head, i) : 0);
    const T* op = reinterpret_cast<const T*>(a.dout) + (live ? a.vdo.row(t.b, head, i) : 0);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[c][s] = load_frag<T>(live ? qp + c * a.vq.sh : nullptr, 16 * s + 8 * hl, a.D);
#pragma unroll
    for (int s = 0; s < VS; ++s) {
      of[s] = load_frag<T>(live ? op : nullptr, 16 * s + 8 * hl, a.Dv);
      if (odd)
#pragma unroll
        for (int j = 0; j < 8; ++j) of[s][j] = -of[s][j];
    }
  }
  float16_t dq[2][DB];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int d = 0; d < DB; ++d) dq[c][d] = zero16();
  // The row's own lift: its lane (and the one of the other half) has all of its dO.
  float norm = 0.f;
  if constexpr (std::is_same<T, half_t>::value) {
#pragma unroll
    for (int s = 0; s < VS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) norm = fmaf((float)of[s][j], (float)of[s][j], norm);
    norm = sqrtf(pair_sum(norm));
  }
  const DsLift<T> lifts(a, t.bh, t.hk, lane);
  const float lift = lifts.of(norm);
  // The rows' common one, for `stat`: the same in every lane, so a scalar register holds it through the sweep.
  const float lift_all = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(lifts.all())));
  const float c2 = a.scale * kLog2e;
  const float lam = live ? a.lam[head * a.lam_step] : 0.f;
  float lse[2], del[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    lse[c] = live ? a.lse[map_at(a, t.b, head, c, i)] : __builtin_inff();
    del[c] = live ? a.delta[map_at(a, t.b, head, c, i)] : 0.f;
  }
  const float d0 = -del[0] * lift, nl = -lam * lift, signed_lift = sign * lift;
  // With what the additions lost: a row's terms one after another would leave some
  // 1e-6 of the sum of thousands. Both together cost 140 -> 144 us (b2 h8 s4096).
  float rest[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};

  // The workgroup goes round together, the last round maybe without a tile for every group.
  for (int first = 0, cur = 0; first < kv_end; first += KG * BN, kv0 += KG * BN, cur ^= 1) {
    wait_copies();
    lds_barrier();
    if (kv0 + KG * BN < kv_end) issue(kv0 + KG * BN, tiles + (cur ^ 1) * kBytes);
    if (kv0 >= own_end) continue;
    const uint32_t tile = tiles + cur * kBytes;
    float16_t p[2], dp = zero16();
    p[0] = p[1] = zero16();
    read_ahead<2 * KS, SH::kDepth>([&](int j) { return KT::row_frag(tile + krow, j % KS, j / KS * kHead); },
                                   [&](int j, frag_t<T> f) { p[j / KS] = Elem<T>::mma(f, qf[j / KS][j % KS], p[j / KS]); });
    read_ahead<VS, SH::kDepth>([&](int s) { return VT::row_frag(tile + vrow, s, 0); },
                               [&](int s, frag_t<T> f) { dp = Elem<T>::mma(f, of[s], dp); });
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int e = 0; e < 16; ++e) p[c][e] = fast_exp2(fmaf(p[c][e], c2, -lse[c]));
      if (kv0 + BN - 1 > free) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (kv0 + acc_row(e, hl) > limit) p[c][e] = 0.f;
      }
    }
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[0][e] *= fmaf(dp[e], signed_lift, d0);
      sum[0] += p[0][e];
      const float u = p[1][e] * fmaf(dp[e], sign, -del[1]);
      sum[1] += u;
      p[1][e] = u * nl;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float y = sum[c] - lost[c], x = rest[c] + y;
      lost[c] = (x - rest[c]) - y;
      rest[c] = x;
    }
    frag_t<T> fs[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int s = 0; s < 2; ++s) fs[c][s] = acc_frag<T>(p[c], s);
    if constexpr (SH::kDepth > 0) __builtin_amdgcn_sched_barrier(0);
    read_ahead<4 * DB, SH::kDepth>(
        [&](int j) { return KT::col_frag(tile + kcol, j % DB, j / (2 * DB) * kHead + 16 * (j / DB % 2) * KT::kRowBytes); },
        [&](int j, frag_t<T> f) {
          const int c = j / (2 * DB), d = j % DB;
          dq[c][d] = Elem<T>::mma(f, fs[c][j / DB % 2], dq[c][d]);
        });
  }

  // The groups' sums, the upper half's added to the lower half's.
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    const int at = (kg % half) * RB + rb;
    float4_t* x = reinterpret_cast<float4_t*>(smem) + at * 2 * DB * 4 * kWave;
    float* y = reinterpret_cast<float*>(smem) + half * RB * 2 * DB * 16 * kWave + at * 2 * kWave;
    __syncthreads();
    if (kg >= half && kg < 2 * half) {
      y[lane] = rest[0];
      y[kWave + lane] = rest[1];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[((c * DB + d) * 4 + e) * kWave + lane] =
                float4_t{dq[c][d][4 * e], dq[c][d][4 * e + 1], dq[c][d][4 * e + 2], dq[c][d][4 * e + 3]};
    }
    __syncthreads();
    if (kg < half) {
      rest[0] += y[lane];
      rest[1] += y[kWave + lane];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float4_t z = x[((c * DB + d) * 4 + e) * kWave + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) dq[c][d][4 * e + j] += z[j];
          }
    }
  }
  if (kg != 0) return;

  rest[0] = pair_sum(rest[0]) / lift;
  rest[1] = pair_sum(rest[1]);
  // P is lifted by pl in its exponent in the dK, dV kernel, and dS by one lift for all
  // rows; what multiplies P to dS takes the former out again.
  const float pl = p_lift<T>(a, t.hk), dl = lift_all / pl;
  if (r >= a.R) return;
  if (hl == 0) {
    a.gsum[row_at(a, t.b, head, i)] = live ? del[1] + rest[1] : 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      *stat_at(a, t.b, head, i, c) = live ? log2f(pl) - lse[c] : -__builtin_inff();
      *stat_at(a, t.b, head, i, 2 + c) = live ? (del[c] + rest[c]) * (c == 0 ? -dl : lam * dl) : 0.f;
    }
  }
  const float out = a.scale / lift;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    T* p = reinterpret_cast<T*>(a.dq) + a.vdq.row(t.b, 2 * head + c, i);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = 32 * d + 8 * e + 4 * hl;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = live ? dq[c][d][4 * e + j] * out : 0.f;
        if (col < a.D) store4t<T>(p + col, y[0], y[1], y[2], y[3]);
      }
  }
}

template <typename T, int HD, int BLOCKS>
int launch_q(DiffArgs a, hipStream_t stream) {
  using SH = QShape<T, HD, BLOCKS>;
  a.n_mtiles = (a.R + 32 * SH::RB - 1) / (32 * SH::RB);
  hipLaunchKernelGGL((diff_bwd_q_kernel<T, HD, BLOCKS>), dim3(uint32_t((int64_t)a.B * a.Hk * a.n_mtiles)),
                     dim3(64 * SH::WAVES), 0, stream, a);
  return tjh::launch_status();
}

// dlam: one workgroup per weight, its rows in a fixed order, in 64 bits. A
// weight for all heads sums [B, H, Sq] from end to end, a head's own B runs of Sq.
__global__ __launch_bounds__(1024) void diff_dlam_kernel(DiffArgs a) {
  __shared__ double red[1024 / kWave];
  const int tid = threadIdx.x, h = blockIdx.x;
  const int64_t run = a.lam_step ? a.Sq : (int64_t)a.B * a.H * a.Sq;
  const int runs = a.lam_step ? a.B : 1;
  double s = 0.;
  for (int b = 0; b < runs; ++b) {
    const float* p = a.gsum + row_at(a, b, h, 0);
    for (int64_t i0 = tid; i0 < run; i0 += 8 * 1024) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = p[min(i0 + 1024 * k, run - 1)];  // no branches: eight loads in flight
#pragma unroll
      for (int k = 0; k < 8; ++k) s += i0 + 1024 * k < run ? x[k] : 0.f;
    }
  }
  for (int m = kWave / 2; m > 0; m >>= 1) s += __shfl_xor(s, m);
  if (tid % kWave == 0) red[tid / kWave] = s;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 1024 / kWave; ++w) s += red[w];
    a.dlam[h] = (float)-s;
  }
}

template <typename T>
int launch_delta(const DiffArgs& a, hipStream_t stream) {
  const int chunks = (a.Dv * (int)sizeof(T) + 15) / 16;
  int lpr = 1;
  while (lpr < chunks) lpr *= 2;
  hipLaunchKernelGGL((diff_delta_kernel<T>), dim3(uint32_t((int64_t)a.n_peaks * a.B * a.Hk)), dim3(kDiffThreads), 0, stream, a, lpr);
  return tjh::launch_status();
}

}  // namespace

int diff_delta(const DiffArgs& a, int dtype, hipStream_t stream) {
  if (dtype == TJ_F32) return launch_delta<float>(a, stream);
  return dtype == TJ_F16 ? launch_delta<half_t>(a, stream) : launch_delta<bf16_t>(a, stream);
}

int diff_bwd_q(const DiffArgs& a, int dtype, hipStream_t stream) {
  const int rc = diff_dispatch(a, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    // 128-row tiles where two workgroups fit a CU: 320 / 360 us (b8 h16 s2048 d64 bf16,
    // 2048 of them). Else 64 rows: 32 dims 184 / 183 us (1024 tiles), 128 dims
    // 329 / 194, 405 / 365, 787 / 725 us (256, 512, 1024 tiles, causal).
    if constexpr (HD == 64 && sizeof(T) == 2)
      if (wide_tiles(a, HD)) return launch_q<T, HD, 4>(a, stream);
    // 32 rows where 64 leave half of the CUs without work, us with 64 / 32: b1 h1 s8192
    // d64 bf16 (128 tiles of 64) 146 / 103, h2 s4096 77 / 56, h8 s1024 25 / 20 (d32: 18 / 12),
    // h12 s1024 (192 tiles) 24.8 / 25.1.
    if constexpr (row_blocks_fit<T, HD>(1))
      if ((int64_t)a.B * a.Hk * ((a.R + 63) / 64) <= kCus / 2) return launch_q<T, HD, 1>(a, stream);
    return launch_q<T, HD, row_blocks_fit<T, HD>(2) ? 2 : 4>(a, stream);
  });
  if (rc != TJ_OK) return rc;
  hipLaunchKernelGGL(diff_dlam_kernel, dim3(a.n_lam), dim3(1024), 0, stream, a);
  return tjh::launch_status();
}

}  // namespace tj
