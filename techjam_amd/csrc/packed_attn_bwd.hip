// Attention of packed sequences with grouped heads, backward (the mathematics, the
// row numbering and the regions are in grouped_attn.h). With the saved row sums,
// P = 2^(scale log2 e S - lse),
//
//   delta = rowsum(dO o O),  dP = dO V^T,  dS = P (dP - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO,
//
// the last two summed over the group's rows. delta comes from the output as it was
// returned plus what its rounding took away, which the forward pass keeps (in bf16
// and fp16; together the two have 16 and 22 bits, in fp16 down to outputs of 2^-14, kRestLift in
// grouped_attn.h): from the rounded output alone dQ and dK
// are 1.55 to 2.4 times as far from 64 bits as one rounding of the result (the most
// for sequences of a few tokens), so 1.45 times. 16-bit inputs have P and dS rounded to
// their type for these products, one rounding more than the result's own (fp32
// MFMAs would take 16 times as long); fp32 inputs have none.
//
// The dQ kernel goes over the keys of its rows and leaves each row's lse and delta
// as the dK, dV kernel wants them; that one goes over the rows of its keys. So
// no atomics are needed, and the result does not depend on the workgroups' order (where several
// share the rows of few keys, their sums are joined in a fixed one); seven
// products a pair are formed where five would do (the others need dQ by atomics).
//
// Medians of a hundred calls after two hundred others. 1904 and 14480 tokens, 16 heads on 8, 128 dims, bf16, causal: dQ
// 1137 us, 1153 TFLOP/s of its three products (the forward kernel 859 us), dK and dV 1648 us, 1060 TFLOP/s of its
// four; matrix units 63 and 56 % busy, vector units 46 and 37, at 1.73 and 1.81 of 2.4 GHz: power, as in the forward kernel (4 % less
// time on another card). 96 sequences of about 340
// tokens, 16 heads on 4, 64 dims: dQ 124 us (of which 79 move rows: 335 MB), dK and dV 138: the first
// 64 keys of the longest, 1870 tokens, have 118 rounds one after the other, 98 us if nothing else runs.
#include <algorithm>

#include "grouped_attn.h"

namespace tj {
namespace {

constexpr int kThreads = 256;
constexpr int kPeakTokens = 64;

// Products with fp16 operands: powers of two that bring the largest possible |dS|,
// 2 |dO_i| |V_j|, near 2^15, so that small gradients and small probabilities keep
// fp16's bits. dQ is a sum over keys, so there every row has its own, by its dO
// (of) and the largest V row of its sequence and key head: a row's bits do not depend on how large the
// gradients of others are. dK sums over rows and has one for all of a (sequence,
// key head), by the largest dO row: dS of a row r times smaller keeps 11 bits down
// to P of about 2^-26 r, and what lies below is off by at most 2^-37 of the largest
// possible |dS|. P itself is lifted by 2^14. 1 for the other types.
template <typename T>
struct DsLift {
  static constexpr bool kOn = std::is_same<T, half_t>::value;
  static constexpr float kP = kOn ? 16384.f : 1.f, kLogP = kOn ? 14.f : 0.f;
  float o = 1.f, v = 1.f;  // the largest norms of dO and V rows
  __device__ __forceinline__ DsLift(const PackedArgs& a, const Region& g, int hk, int lane) {
    if constexpr (kOn) {
      const float* pk = a.peak + ((int64_t)Region::slot(g.start, g.index, 1, kPeakTokens) * a.Hk + hk) * 2;
      o = v = 0.f;
      for (int s = lane; s * kPeakTokens < g.len; s += kWave) {
        o = fmaxf(o, pk[(int64_t)s * a.Hk * 2]);
        v = fmaxf(v, pk[(int64_t)s * a.Hk * 2 + 1]);
      }
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) {
        o = fmaxf(o, __shfl_xor(o, m));
        v = fmaxf(v, __shfl_xor(v, m));
      }
    }
  }
  // For rows whose dO has at most this norm.
  __device__ __forceinline__ float of(float norm) const {
    if constexpr (!kOn) return 1.f;
    // Exponents rather than products: the norms' product may leave fp32.
    int ex, ey;
    frexpf(norm, &ex);
    frexpf(v, &ey);
    if (!(norm > 0.f) || !(norm < 3e38f) || !(v > 0.f)) return 1.f;  // a row that is not finite is lost anyway
    return ldexpf(1.f, min(max(14 - ex - ey, -100), 100));
  }
  // Of all rows: the same in every lane, so a scalar register holds it.
  __device__ __forceinline__ float all() const {
    return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(of(o))));
  }
};

// The largest norms of 64 tokens' dO rows (all heads of the group) and V rows, those that are finite: others
// spoil their own row only. A group of `lpr` lanes a row, 16-byte chunks.
__global__ __launch_bounds__(kThreads) void packed_peak_kernel(PackedArgs a, int lpr) {
  __shared__ float red[2][kThreads / kWave];
  const int tid = threadIdx.x, hk = blockIdx.x % a.Hk, at = blockIdx.x / a.Hk;
  Region g;
  if (!g.find(a, at, 1, kPeakTokens, tid % kWave)) return;
  const int lane = tid % lpr, per_block = kThreads / lpr, first = g.tile * kPeakTokens;
  const int tokens = min(kPeakTokens, g.len - first);
  const bool on = lane * 8 < a.Dv;
  auto norm2 = [&](const half_t* p) {
    float n = 0.f;
    if (on) {
      const half8_t x = *reinterpret_cast<const half8_t*>(p + lane * 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) n = fmaf((float)x[e], (float)x[e], n);
    }
    for (int s = lpr / 2; s > 0; s >>= 1) n += __shfl_xor(n, s);
    return n < 3e38f ? n : 0.f;
  };
  float peak[2] = {0.f, 0.f};
  for (int r = tid / lpr; r < tokens * a.G; r += per_block)
    peak[0] = fmaxf(peak[0], norm2(reinterpret_cast<const half_t*>(a.dout) +
                                   a.vdo.row(g.start + first + r / a.by_group, hk * a.G + r % a.by_group)));
  for (int j = tid / lpr; j < tokens; j += per_block)
    peak[1] = fmaxf(peak[1], norm2(reinterpret_cast<const half_t*>(a.v) + a.vv.row(g.start + first + j, hk)));
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    for (int s = kWave / 2; s > 0; s >>= 1) peak[c] = fmaxf(peak[c], __shfl_xor(peak[c], s));
    if (tid % kWave == 0) red[c][tid / kWave] = peak[c];
  }
  __syncthreads();
  if (tid < 2) {
    float x = red[tid][0];
    for (int w = 1; w < kThreads / kWave; ++w) x = fmaxf(x, red[tid][w]);
    a.peak[((int64_t)at * a.Hk + hk) * 2 + tid] = sqrtf(x);
  }
}

// The numbers of 32 tokens of a head: 32 of log2(lift of P) - lse, 32 of -delta, lifted.
__device__ __forceinline__ float* stat_at(const PackedArgs& a, const Region& g, int head, int i) {
  return a.stat + (((int64_t)Region::slot(g.start, g.index, 1, 32) + i / 32) * a.H + head) * 64 + i % 32;
}

// A workgroup = RB waves of 32 rows times KG groups, keys through LDS in
// tiles of 32 or 64 dealt to the groups in turn, whose sums meet in LDS at the end. Scores
// transposed as in the forward kernel: a row's sums are its lane's own numbers, and
// dS turns into the B operand of dQ^T = K^T dS^T.
template <typename T, int HD, int BLOCKS>
struct QShape {
  static constexpr int RB = BLOCKS, KG = 4 / RB, ROWS = 32 * RB;
  static constexpr int BN = KG == 1 && HD * (int)sizeof(T) <= 256 ? 64 : 32;  // half the meetings: 1170 -> 1145 us (128 dims), 143 -> 132 (64)
  using SH = SweepShape<T, HD, BN>;
  using Wave = WaveRows<T, HD>;
  // Two tiles a group, afterwards the groups' sums. The rows come through the second tile while the first keys are on
  // their way, or through a place of their own where it has no room for them.
  static constexpr int kTiles = KG * 2 * SH::kBytes, kSums = KG > 1 ? KG / 2 * RB * SH::DB * 16 * kWave * 4 : 0;
  static constexpr bool kOwn = RB * Wave::kBytes > SH::kBytes;
  static constexpr int kWithRows = kTiles + (kOwn ? RB * Wave::kBytes : 0), kBytes = kWithRows > kSums ? kWithRows : kSums;
  static_assert(!kOwn || KG == 1, "places are one group's");
};
template <typename T, int HD>
constexpr bool groups_fit(int groups) { return groups * SweepShape<T, HD, 32>::W * (int)sizeof(T) <= 1024; }

template <typename T, int HD, int BLOCKS>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 2 && HD <= 64 ? 3 : (HD * (int)sizeof(T) <= 256 ? 2 : 1))) void packed_bwd_q_kernel(PackedArgs a) {
  using QS = QShape<T, HD, BLOCKS>;
  using SH = typename QS::SH;
  using Wave = typename QS::Wave;
  using Rows = typename SH::Rows;
  constexpr int KS = SH::KS, DB = SH::DB, BN = QS::BN, RB = QS::RB, KG = QS::KG, ROWS = QS::ROWS, kDepth = SH::kDepth;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[QS::kBytes];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, hl = lane / 32;
  const int kg = w / RB, rb = w % RB, hk = blockIdx.x % a.Hk;
  __shared__ int told[6];
  Region g;
  if (!g.take(a, blockIdx.x / a.Hk, a.G, ROWS, false, tid, told)) return;
  const int L = g.len, R = g.rows * a.G, r0 = g.tile * ROWS, rw0 = r0 + 32 * rb;
  auto span = [&](int row, int last) {
    return row >= R || row / a.by_group >= L ? 0 : (a.causal ? min(L, min(last, R - 1) / a.by_group + 1) : L);
  };
  const int kv_end = span(r0, r0 + ROWS - 1), own_end = span(rw0, rw0 + 31);
  const uint32_t tiles = lds_offset(smem) + kg * 2 * SH::kBytes;
  const uint32_t krow = Rows::lane_row(lane), kcol = Rows::lane_col(lane), vrow = krow + SH::kTensor;
  SweepTiles<T, SH, RB> keys;
  keys.init(reinterpret_cast<const T*>(a.k) + a.vk.row(g.start, hk), reinterpret_cast<const T*>(a.v) + a.vv.row(g.start, hk),
            a.vk.st, a.vv.st, a.D, a.Dv, rb, lane);
  int kv0 = BN * kg;
  if (kv0 < kv_end) keys.issue(kv0, L, tiles, rb);

  const int r = rw0 + lane % 32;
  SweepRow row{r / a.by_group, r % a.by_group, 0, r < R && r / a.by_group < L};
  row.limit = a.causal ? row.i : L - 1;
  const int free = a.causal ? rw0 / a.by_group : L - 1;  // the last key that all of the wave's rows see
  const typename Wave::Places places(rw0, a.by_group, lane);
  const int64_t token0 = g.start + rw0 / a.by_group;
  frag_t<T> qf[KS], of[KS];
  float sum = 0.f, norm = 0.f;
  {
    typename Wave::vec_t xq[Wave::N], xo[Wave::N], xy[Wave::N], xz[Wave::N];
    const int end = L * a.G;
    const int64_t at = a.vo.row(token0, hk * a.G);
    Wave::read(xq, reinterpret_cast<const T*>(a.q) + a.vq.row(token0, hk * a.G), a.vq.st, a.vq.sh, a.D, places, end, lane);
    Wave::read(xo, reinterpret_cast<const T*>(a.dout) + a.vdo.row(token0, hk * a.G), a.vdo.st, a.vdo.sh, a.Dv, places, end, lane);
    Wave::read(xy, reinterpret_cast<const T*>(a.out) + at, a.vo.st, a.vo.sh, a.Dv, places, end, lane);
    if constexpr (sizeof(T) == 2) Wave::read(xz, reinterpret_cast<const T*>(a.rest) + at, a.vo.st, a.vo.sh, a.Dv, places, end, lane);
    const uint32_t turn = QS::kOwn ? lds_offset(smem) + QS::kTiles + rb * Wave::kBytes : tiles + SH::kBytes + rb * Wave::kBytes;
    frag_t<T> y[KS];
    auto dot = [&](float x) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x = fmaf((float)of[s][j], (float)y[s][j], x);
      return x;
    };
    Wave::turn(xq, turn, lane, qf);
    Wave::turn(xo, turn, lane, of);
    Wave::turn(xy, turn, lane, y);
    sum = dot(0.f);
    if constexpr (sizeof(T) == 2) {
      Wave::turn(xz, turn, lane, y);
      sum = kRestLift<T> == 1.f ? dot(sum) : fmaf(dot(0.f), 1.f / kRestLift<T>, sum);
    }
  }
  float del = pair_sum(sum);
  const float lse = row.live ? a.lse[(int64_t)(g.start + row.i) * a.H + hk * a.G + row.g] : __builtin_inff();
  // The row's own lift: its lane (and the one of the other half) has all of its dO.
  const DsLift<T> lifts(a, g, hk, lane);
  float lift = 1.f;
  if constexpr (DsLift<T>::kOn) {
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) norm = fmaf((float)of[s][j], (float)of[s][j], norm);
    lift = lifts.of(sqrtf(pair_sum(norm)));
  }
  const float common = lifts.all() / DsLift<T>::kP, c2 = a.scale * kLog2e;
  float d0 = -del * lift;
  float16_t dq[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dq[d] = zero16();

  // The workgroup goes round together, the last round maybe without a tile for every group.
  for (int first = 0, cur = 0; first < kv_end; first += KG * BN, kv0 += KG * BN, cur ^= 1) {
    wait_copies();
    lds_barrier();
    if (kv0 + KG * BN < kv_end) keys.issue(kv0 + KG * BN, L, tiles + (cur ^ 1) * SH::kBytes, rb);
    const uint32_t tile = tiles + cur * SH::kBytes;
#pragma unroll
    for (int kb = 0; kb < BN / 32; ++kb) {
      const int at = kv0 + 32 * kb;
      if (at < own_end) {
        const int rows = kb * 32 * Rows::kRowBytes;
        float16_t p = zero16(), dp = zero16();
        read_ahead<2 * KS, kDepth>([&](int s) { return Rows::row_frag(tile + (s < KS ? krow : vrow), s % KS, rows); },
                                   [&](int s, frag_t<T> f) {
                                     if (s < KS) p = Elem<T>::mma(f, qf[s % KS], p);
                                     else dp = Elem<T>::mma(f, of[s % KS], dp);
                                   });
        if (own_end <= 32) {
          // Rows of 32 keys: delta = sum of P dP, exact to what fp32 sums are. (The output's has the rounding of P in it, which
          // shows where few keys share a row: sequences of two tokens, dQ 1.4 instead of 1.6 times one rounding from 64 bits.)
          float exact = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at + acc_row(e, hl) <= row.limit) exact = fmaf(fast_exp2(fmaf(p[e], c2, -lse)), dp[e], exact);
          del = pair_sum(exact);
          d0 = -del * lift;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = fast_exp2(fmaf(p[e], c2, -lse)) * fmaf(dp[e], lift, d0);
        // Selected, not multiplied: what a masked key holds does not matter.
        if (at + 31 > free) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at + acc_row(e, hl) > row.limit) p[e] = 0.f;
        }
        frag_t<T> fs[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) fs[s] = acc_frag<T>(p, s);
        if constexpr (kDepth > 0) __builtin_amdgcn_sched_barrier(0);
        read_ahead<2 * DB, kDepth>(
            [&](int j) { return Rows::col_frag(tile + kcol, j % DB, rows + 16 * (j / DB) * Rows::kRowBytes); },
            [&](int j, frag_t<T> f) { dq[j % DB] = Elem<T>::mma(f, fs[j / DB], dq[j % DB]); });
      }
    }
  }

  // The groups' sums, the upper half's added to the lower half's.
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    float4_t* x = reinterpret_cast<float4_t*>(smem) + ((kg % half) * RB + rb) * DB * 4 * kWave + lane;
    __syncthreads();
    if (kg >= half && kg < 2 * half) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[(d * 4 + e) * kWave] = float4_t{dq[d][4 * e], dq[d][4 * e + 1], dq[d][4 * e + 2], dq[d][4 * e + 3]};
    }
    __syncthreads();
    if (kg < half) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4_t z = x[(d * 4 + e) * kWave];
#pragma unroll
          for (int j = 0; j < 4; ++j) dq[d][4 * e + j] += z[j];
        }
    }
  }
  __syncthreads();  // the tiles, in whose place the rows are turned, have been read
  if (kg != 0) return;

  if (row.live && hl == 0) {
    float* st = stat_at(a, g, hk * a.G + row.g, row.i);
    st[0] = DsLift<T>::kLogP - lse;
    st[32] = -del * common;
  }
  const float out = a.scale / lift;
  Wave::write(reinterpret_cast<T*>(a.dq) + a.vdq.row(token0, hk * a.G), a.vdq.st, a.vdq.sh, a.D, places, R,
              lds_offset(smem) + rb * Wave::kBytes, lane, [&](int d, int c) {
                float4_t y = {0.f, 0.f, 0.f, 0.f};
                if (row.live) y = float4_t{dq[d][4 * c], dq[d][4 * c + 1], dq[d][4 * c + 2], dq[d][4 * c + 3]} * out;
                return y;
              });
}

// A workgroup = KB waves of 32 keys of one (sequence, key head) times RG
// groups of token tiles: the tiles of 32 tokens that see the keys, of one query
// head of the group after the other, are dealt to the groups in turn, and the
// groups' sums meet in LDS at the end. Scores are formed with tokens in the
// registers and keys over the lanes, so that P and dS turn into the A operands of dV
// and dK where they stand; Q and dO come back as B operands through the transposing
// LDS read.
template <typename T, int HD, int BLOCKS, int GROUPS>
struct KvShape {
  using SH = SweepShape<T, HD, 32>;
  static constexpr int KB = BLOCKS, RG = GROUPS, WAVES = KB * RG, KEYS = 32 * KB;
  // 64 dims: 142 us with two, 139 with three; 128 dims: 1629 and 1669.
  static constexpr int kDepth = HD == 32 ? 0 : sizeof(T) == 2 ? (HD == 64 ? 3 : 2) : 1;
  // Waves of a SIMD, by the registers: with one at 128 dims (310 registers) 2534 us instead of 1600, with two at 64
  // dims 37 instead of 28.
  static constexpr int kMin = sizeof(T) == 2 ? (HD <= 64 && KB > 1 ? 3 : 2) : (HD == 32 ? 2 : 1);
};

template <typename T, int HD, int BLOCKS, int GROUPS>
__global__ __launch_bounds__((64 * BLOCKS * GROUPS), (KvShape<T, HD, BLOCKS, GROUPS>::kMin)) void
packed_bwd_kv_kernel(PackedArgs a) {
  using KV = KvShape<T, HD, BLOCKS, GROUPS>;
  using SH = typename KV::SH;
  using Rows = typename SH::Rows;
  constexpr int KS = SH::KS, DB = SH::DB, BM = 32, KB = KV::KB, RG = KV::RG, kDepth = KV::kDepth;
  constexpr int kSums = RG / 2 * KB * 2 * DB * 16 * kWave * 4;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[RG * 2 * SH::kBytes > kSums ? RG * 2 * SH::kBytes : kSums];  // Q's tile, then dO's
  __shared__ __attribute__((aligned(1024))) float stat[RG][2][64];  // of a tile's tokens
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, hl = lane / 32,
            ln = lane % 32;
  const int kb = w % KB, rg = w / KB, hk = blockIdx.x % a.Hk;
  __shared__ int told[6];
  Region g;
  const int share = blockIdx.x / a.Hk % a.shares;
  if (!g.take(a, blockIdx.x / a.Hk / a.shares, 1, KV::KEYS, true, tid, told)) return;
  const int L = g.len, k0 = g.tile * KV::KEYS, kw0 = k0 + 32 * kb, key = kw0 + ln;

  // The group's KB waves bring its tiles.
  SweepTiles<T, SH, KB> rows;
  rows.init(nullptr, nullptr, a.vq.st, a.vdo.st, a.D, a.Dv, kb, lane);
  const T* qp = reinterpret_cast<const T*>(a.q) + a.vq.row(g.start, hk * a.G);
  const T* op = reinterpret_cast<const T*>(a.dout) + a.vdo.row(g.start, hk * a.G);
  const uint32_t group = lds_offset(smem) + rg * 2 * SH::kBytes, stat0 = lds_offset(stat[rg]);
  const uint32_t qrow = Rows::lane_row(lane), qcol = Rows::lane_col(lane), orow = qrow + SH::kTensor, ocol = qcol + SH::kTensor;
  // Tile n: head n / tiles of the group, tokens i_begin + 32 (n % tiles) on. They are dealt to the groups of all
  // workgroups that share the keys.
  const int i_begin = a.causal ? k0 : 0;
  const int tiles = k0 < L ? (L - i_begin + BM - 1) / BM : 0, n_end = tiles * a.G;
  // `n` tiles further on: the head and the token (no division in the loop).
  auto advance = [&](int& h, int& i0, int n) {
    i0 += BM * n;
    while (i0 >= i_begin + BM * tiles) {
      i0 -= BM * tiles;
      ++h;
    }
  };
  auto issue = [&](int h, int i0, int buf) {
    rows.kp = qp + h * a.vq.sh;
    rows.vp = op + h * a.vdo.sh;
    rows.issue(i0, L, group + buf * SH::kBytes, kb);
    // The tokens' numbers by the same way: a load into registers would have to be waited for,
    // and every copy issued before with it.
    if (kb == 0) copy_4(make_rsrc(stat_at(a, g, hk * a.G + h, i0), 256), stat0 + buf * 256, 4 * lane);
  };

  int h = 0, i0 = i_begin;  // this round's tile
  const int n0 = share * RG + rg, step = a.shares * RG;
  if (n0 < n_end) {
    advance(h, i0, n0);
    issue(h, i0, 0);
  }
  frag_t<T> kf[KS], vf[KS];
  {
    // Through the second tile, while the first is on its way.
    using Wave = WaveRows<T, HD>;
    static_assert(KB * Wave::kBytes <= SH::kBytes, "room for the keys");
    typename Wave::vec_t xk[Wave::N], xv[Wave::N];
    const typename Wave::Places places(kw0, Divisor{1u << 31, 0, 1}, lane);  // a group of one
    Wave::read(xk, reinterpret_cast<const T*>(a.k) + a.vk.row(g.start + kw0, hk), a.vk.st, 0, a.D, places, L, lane);
    Wave::read(xv, reinterpret_cast<const T*>(a.v) + a.vv.row(g.start + kw0, hk), a.vv.st, 0, a.Dv, places, L, lane);
    Wave::turn(xk, group + SH::kBytes + kb * Wave::kBytes, lane, kf);
    Wave::turn(xv, group + SH::kBytes + kb * Wave::kBytes, lane, vf);
  }
  float16_t dv[DB], dk[DB];
#pragma unroll
  for (int d = 0; d < DB; ++d) dv[d] = dk[d] = zero16();

  const float dl = DsLift<T>(a, g, hk, lane).all(), lift = dl / DsLift<T>::kP, c2 = a.scale * kLog2e;
  // The workgroup goes round together, the last round maybe without a tile for every group.
  const int rounds = (n_end - share * RG + step - 1) / step;
  for (int round = 0, n = n0, cur = 0; round < rounds; ++round, n += step, cur ^= 1) {
    // The tile is there, and the group's other one has been read by its waves.
    wait_copies();
    lds_barrier();
    const uint32_t tile = group + cur * SH::kBytes, srow = stat0 + cur * 256 + 16 * hl;
    // Else there is no tile, or every token stands before the wave's keys.
    const bool busy = n < n_end && (!a.causal || i0 + BM > kw0);
    const int at = i0;
    if (n + step < n_end) {
      advance(h, i0, step);
      issue(h, i0, cur ^ 1);
    }
    if (!busy) continue;
    float16_t p = zero16(), dp = zero16();
    read_ahead<2 * KS, kDepth>([&](int s) { return Rows::row_frag(tile + (s < KS ? qrow : orow), s % KS, 0); },
                               [&](int s, frag_t<T> f) {
                                 if (s < KS) p = Elem<T>::mma(f, kf[s % KS], p);
                                 else dp = Elem<T>::mma(f, vf[s % KS], dp);
                               });
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4_t ls = lds_at<float4_t>(srow + q * 32), d0 = lds_at<float4_t>(srow + 128 + q * 32);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = fast_exp2(fmaf(p[4 * q + j], c2, ls[j]));
        p[4 * q + j] = e;
        dp[4 * q + j] = e * fmaf(dp[4 * q + j], lift, d0[j]);
      }
    }
    // Selected, not multiplied: tokens past the length have no numbers at all.
    if ((a.causal && at < kw0 + 31) || at + BM > L) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = at + acc_row(r, hl);
        if ((a.causal && i < key) || i >= L) p[r] = dp[r] = 0.f;
      }
    }
    frag_t<T> fp[2], fs[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      fp[s] = acc_frag<T>(p, s);
      fs[s] = acc_frag<T>(dp, s);
    }
    if constexpr (kDepth > 0) __builtin_amdgcn_sched_barrier(0);
    read_ahead<4 * DB, kDepth>(
        [&](int j) { return Rows::col_frag(tile + (j < 2 * DB ? ocol : qcol), j % DB, 16 * (j / DB % 2) * Rows::kRowBytes); },
        [&](int j, frag_t<T> f) {
          if (j < 2 * DB) dv[j % DB] = Elem<T>::mma(fp[j / DB % 2], f, dv[j % DB]);
          else dk[j % DB] = Elem<T>::mma(fs[j / DB % 2], f, dk[j % DB]);
        });
  }

  // The groups' sums, the upper half's added to the lower half's.
  if constexpr (RG > 1) {
    auto each = [&](auto&& f) {
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        f(dv[d], 2 * d);
        f(dk[d], 2 * d + 1);
      }
    };
#pragma unroll
    for (int half = RG / 2; half > 0; half /= 2) {
      float4_t* y = reinterpret_cast<float4_t*>(smem) + ((rg % half) * KB + kb) * 2 * DB * 4 * kWave + lane;
      __syncthreads();
      if (rg >= half && rg < 2 * half)
        each([&](float16_t& x, int i) {
#pragma unroll
          for (int q = 0; q < 4; ++q) y[(4 * i + q) * kWave] = float4_t{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
        });
      __syncthreads();
      if (rg < half)
        each([&](float16_t& x, int i) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4_t z = y[(4 * i + q) * kWave];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * q + j] += z[j];
          }
        });
    }
    if (rg != 0) return;
  }

  // Keys at or past the length have no gradient: zeros, whatever their scores were.
  const float dv_scale = 1.f / DsLift<T>::kP, dk_scale = a.scale / dl;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = kw0 + acc_row(r, hl);
    if (j >= g.rows) continue;
    const bool in = j < L;
    if (a.shares > 1) {
      float* x = a.part + (((int64_t)share * a.T + g.start + j) * a.Hk + hk) * (a.Dv + a.D);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        if (32 * d + ln < a.Dv) x[32 * d + ln] = in ? dv[d][r] * dv_scale : 0.f;
        if (32 * d + ln < a.D) x[a.Dv + 32 * d + ln] = in ? dk[d][r] * dk_scale : 0.f;
      }
      continue;
    }
    T* pv = reinterpret_cast<T*>(a.dv) + a.vdv.row(g.start + j, hk);
    T* pk = reinterpret_cast<T*>(a.dk) + a.vdk.row(g.start + j, hk);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      if (32 * d + ln < a.Dv) pv[32 * d + ln] = (T)(in ? dv[d][r] * dv_scale : 0.f);
      if (32 * d + ln < a.D) pk[32 * d + ln] = (T)(in ? dk[d][r] * dk_scale : 0.f);
    }
  }
}

// dV and dK of the workgroups that shared the rows of a key tile, summed in their order; four columns a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void packed_bwd_join_kernel(PackedArgs a) {
  const int width = a.Dv + a.D, chunks = width / 4;
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x, row = at / chunks;
  if (row >= (int64_t)a.T * a.Hk) return;
  const int col = (int)(at - row * chunks) * 4, hk = (int)(row % a.Hk);
  const int64_t t = row / a.Hk, step = (int64_t)a.T * a.Hk * width;
  const float* x = a.part + row * width + col;
  float4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.shares; ++s) y += *reinterpret_cast<const float4_t*>(x + s * step);
  T* p = col < a.Dv ? reinterpret_cast<T*>(a.dv) + a.vdv.row(t, hk) + col : reinterpret_cast<T*>(a.dk) + a.vdk.row(t, hk) + col - a.Dv;
  store4t<T>(p, y[0], y[1], y[2], y[3]);
}

template <typename T, int HD, int BLOCKS>
int launch_q(PackedArgs a, hipStream_t stream) {
  const int64_t slots = region_slots(a.T, a.N, a.G, QShape<T, HD, BLOCKS>::ROWS);
  a.n_slots = (int)slots;
  hipLaunchKernelGGL((packed_bwd_q_kernel<T, HD, BLOCKS>), dim3(uint32_t(slots * a.Hk)), dim3(kThreads), 0, stream, a);
  return tjh::launch_status();
}

template <typename T, int HD, int BLOCKS, int GROUPS>
int launch_kv(PackedArgs a, hipStream_t stream) {
  using KV = KvShape<T, HD, BLOCKS, GROUPS>;
  const int64_t slots = region_slots(a.T, a.N, 1, KV::KEYS);
  a.n_slots = (int)slots;
  hipLaunchKernelGGL((packed_bwd_kv_kernel<T, HD, BLOCKS, GROUPS>), dim3(uint32_t(slots * a.Hk * a.shares)), dim3(64 * KV::WAVES), 0,
                     stream, a);
  const int rc = tjh::launch_status();
  if (rc != TJ_OK || a.shares == 1) return rc;
  const int64_t chunks = (int64_t)a.T * a.Hk * ((a.Dv + a.D) / 4);
  hipLaunchKernelGGL((packed_bwd_join_kernel<T>), dim3(uint32_t((chunks + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, a);
  return tjh::launch_status();
}

}  // namespace

// Key tiles are few where few key heads serve many query heads, and each then has many rounds, 0.85 us apiece at 64
// dims whatever else runs: with 256 workgroups of them the dK, dV kernel took 437 us beside 115 of dQ (4096 tokens, 32
// heads on 4). So several workgroups share a tile's rows, up to 1024 in all and 16 rounds each or more of a sequence of
// ordinary length; their sums go through memory. us with one / two / four / eight, joining included, bf16: 4096 tokens, 32
// heads on 4, 64 dims (256 tiles) 440 / 262 / 169 / 181; 4 x 2048, 16 on 2, 128 dims (256) 319 / 202 / 177 / 202; 4096,
// 32 on 8, 128 dims (512) 356 / 313 / 332 / 411; 8192, 32 on 8, 128 dims (1024) 1091 / 1065 / 1120 / 1267; 2048, 16 on 2, 64
// dims (64) with four / twelve / sixteen 70 / 40 / 42 instead of 120. Rounds of fp32 take about six times as long and half as many
// workgroups fill the chip: 512 and four rounds. us with one / two / four / eight: 2000 tokens, 2 on 2, 96 dims (64
// tiles) 212 / 120 / 71 / 66; 2 x 700, 8 on 8, 64 dims (176) 62 / 53 / 75 / 116; 2 x 2000, 16 on 4, 128 dims (252)
// 1056 / 621 / 651 / 729; 1024, 4 on 4, 64 dims (64) 51 / 54 / 38 / 47.
int packed_bwd_shares(int dtype, int64_t T, int64_t N, int64_t H, int64_t Hk) {
  const int64_t tiles = std::max<int64_t>(1, (T + 63) / 64 * Hk);
  const int64_t rounds = (T / std::max<int64_t>(N, 1) + 31) / 32 * (H / Hk) / 2;
  const bool wide = dtype == TJ_F32;
  const int64_t shares = std::max<int64_t>(1, std::min<int64_t>({16, (wide ? 512 : 1024) / tiles, rounds / (wide ? 4 : 16)}));
  // Four groups of a workgroup with 32 keys do what two workgroups would: 120 us and 116 + 4.
  return shares == 2 && !wide && tiles <= kCus / 2 ? 1 : (int)shares;
}

int packed_bwd(const PackedArgs& a, int dtype, hipStream_t stream) {
  if (dtype == TJ_F16) {
    int lpr = 1;
    while (lpr * 8 < a.Dv) lpr *= 2;
    const int64_t slots = region_slots(a.T, a.N, 1, kPeakTokens);
    hipLaunchKernelGGL(packed_peak_kernel, dim3(uint32_t(slots * a.Hk)), dim3(kThreads), 0, stream, a, lpr);
    if (const int rc = tjh::launch_status()) return rc;
  }
  return grouped_dispatch(a.D, a.Dv, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    const int64_t rows = (int64_t)a.T * a.G;  // of one key head
    // us with 128 / 64 rows a workgroup: 512 tiles of 128 rows, 64 dims 31 / 22; 4260 tiles 137 / 187; 2056 tiles of 128 dims
    // 1142 / 1248; 768 tiles of 64 dims of a causal sequence of 16384 382 / 347, 1024 of 512 tokens 37 / 41.
    const int64_t most = (HD <= 64 && sizeof(T) == 2 && long_triangles(a) ? 3 : 2) * kCus;
    int rc;
    if constexpr (groups_fit<T, HD>(4)) {
      if ((rows + 63) / 64 * a.Hk <= kCus / 2) rc = launch_q<T, HD, 1>(a, stream);
      else if ((rows + 127) / 128 * a.Hk <= most) rc = launch_q<T, HD, 2>(a, stream);
      else rc = launch_q<T, HD, 4>(a, stream);
    } else {
      if ((rows + 127) / 128 * a.Hk <= most) rc = launch_q<T, HD, 2>(a, stream);
      else rc = launch_q<T, HD, 4>(a, stream);
    }
    if (rc != TJ_OK) return rc;
    // 64 keys, or 32 where those leave half of the CUs idle. us with 128 / 64 / 32 keys a workgroup: short sequences of 64 dims
    // 298 / 234 / 266, long ones of 128 dims 1589 / 1601 / 2439.
    if (a.shares == 1 && (int64_t)(a.T + 63) / 64 * a.Hk <= kCus / 2) return launch_kv<T, HD, 1, groups_fit<T, HD>(4) ? 4 : 2>(a, stream);
    return launch_kv<T, HD, 2, 2>(a, stream);
  });
}

}  // namespace tj
