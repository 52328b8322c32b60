// Differential attention, forward (the mathematics and the row numbering are
// in diff_attn.h): whole sequences, and few new tokens against a cache.
//
// Scores are formed transposed, S^T = K Q^T, so that a lane holds scores of ONE
// row: maximum and sum are per lane (the other half of the wave holds the
// other keys), and the probabilities turn into the B operand of O^T = V^T P^T
// where they stand. The two maps have their own running maximum, sum and
// accumulator and share every V fragment.
//
// diff_fwd_kernel: a workgroup = RB blocks of 32 rows of one (b, key head) times
// KG groups, a wave each; key tiles of 32 or 64 stream through LDS, dealt to the
// groups in turn, and the groups' sums meet in LDS at the end. diff_few_kernel: a
// workgroup = one wave = 32 rows and one part of the keys, with its own LDS tile.
// Sweeps cut into parts are joined by diff_join_kernel.
//
// Long sequences are bound by the matrix and vector units together: b2 h8 s8192
// d64 bf16 causal takes 425 us, 970 TFLOP/s of its own 4D + 4Dv operations a pair
// (a large library product of that type runs at 1144), matrix units busy 53 % and
// vector units 58 % of the time, no LDS bank conflicts. Few rows are bound by the
// cache's bytes: 16 sequences of 16384 to 65536 keys, 4 key heads, d64 bf16, one
// token: 240 us + 7 us of joining, 5.6 TB/s (a copy of 1 GiB: 5.1).
#include "diff_attn.h"

namespace tj {
namespace {

constexpr float kLazy = 8.f;  // the running maximum moves when a row's maximum grows by more than 2^8

template <typename T, int HD, int BNT>
struct FwdShape {
  static constexpr int DVP = 2 * HD;
  static constexpr int BN = BNT;  // keys of a tile
  using KT = LdsRows<T, HD>;
  using VT = LdsRows<T, DVP>;
  static constexpr int KS = HD / 16;   // k-steps over the head dim
  static constexpr int DB = DVP / 32;  // output blocks
  // Operands read ahead where the registers have room (us without / with): 128 dims,
  // 186 / 174 and 154 / 141 (b2 h4 s4096 causal bf16, 128- and 64-row tiles), 64 dims in
  // tiles of 64 keys 515 / 502 (b4 h16 s4096); in those of 32 it costs,
  // 168 / 175, and so it does in fp32, 452 / 475 (b2 h4 s2048 d128).
  static constexpr int kDepth = sizeof(T) == 2 && (HD == 128 || (HD == 64 && BN > 32)) ? 2 : 0;
  static constexpr int kElems = BN * (2 * HD + DVP);  // one tile of both key heads and of V
  static constexpr int kBytes = kElems * (int)sizeof(T), kHead = BN * HD * (int)sizeof(T);
};

// A lane's row: r of the (b, key head), its token, head and position, and the last key it sees.
struct DiffRow {
  int r, i, g, limit;
  bool live;
  __device__ __forceinline__ DiffRow(const DiffArgs& a, int row, int L) : r(row), i(row / a.G), g(row % a.G) {
    const int pos = (a.cached ? L - a.Sq : 0) + i;
    live = r < a.R && pos >= 0 && pos < L;
    limit = a.causal ? pos : L - 1;
  }
};

// Rows row0 .. row1 (clipped to R) of a wave or workgroup: keys needed, and the
// last key that every one of them sees.
struct DiffSpan {
  int end, free;
  __device__ __forceinline__ DiffSpan(const DiffArgs& a, int row0, int row1, int L) {
    const int first = a.cached ? L - a.Sq : 0;
    const int p0 = first + row0 / a.G, p1 = first + min(row1, a.R - 1) / a.G;
    end = row0 >= a.R || p0 >= L || p1 < 0 ? 0 : (a.causal ? min(L, p1 + 1) : L);
    free = a.causal ? p0 : L - 1;
  }
};

// The running state of a wave's 32 rows, for NM maps from map `first` on: both,
// or one where two accumulators of the width exceed a wave's registers (a pair
// of waves then shares the rows and the key tiles).
// The output is divided by the sum of the probabilities as they were rounded for
// its product (to the inputs' type: fp32 MFMAs would take 16 times as long): a dominant key's rounding cancels, and two go into one
// instruction. What the backward pass gets (STATS) is the sum of the unrounded
// ones, so that its P sums to 1 as exactly as fp32 does.
template <typename T, int HD, int BN, int NM, bool STATS>
struct FwdState {
  using SH = FwdShape<T, HD, BN>;
  frag_t<T> q[NM][SH::KS];
  float16_t o[NM][SH::DB];
  float m[NM], l[NM];  // maximum in log2 units, the lane's part of the sum
  float e[STATS ? NM : 1];
  float c2;            // |scale| log2 e
  int first;
  uint32_t kbase, vbase;  // the lane's places in a key tile

  __device__ __forceinline__ void init(const DiffArgs& a, int b, int hk, const DiffRow& row, int first_map, int lane) {
    const int hl = lane / 32;
    first = first_map;
    kbase = SH::KT::lane_row(lane) + first * SH::kHead;
    vbase = SH::VT::lane_col(lane) + 2 * SH::kHead;
    const T* qp = reinterpret_cast<const T*>(a.q) + (row.live ? a.vq.row(b, 2 * (hk * a.G + row.g), row.i) : 0);
    // A negative scale turns q's sign, so that the largest score is the largest
    // product; a zero one becomes too small to matter, so that masked stays -inf.
    c2 = fmaxf(fabsf(a.scale) * kLog2e, 1e-37f);
#pragma unroll
    for (int c = 0; c < NM; ++c) {
#pragma unroll
      for (int ks = 0; ks < SH::KS; ++ks) {
        q[c][ks] = load_frag<T>(row.live ? qp + (first + c) * a.vq.sh : nullptr, 16 * ks + 8 * hl, a.D);
        if (a.scale < 0.f)
#pragma unroll
          for (int j = 0; j < 8; ++j) q[c][ks][j] = -q[c][ks][j];
      }
      m[c] = -__builtin_inff();
      l[c] = 0.f;
      if constexpr (STATS) e[c] = 0.f;
#pragma unroll
      for (int d = 0; d < SH::DB; ++d) o[c][d] = zero16();
    }
  }

  // 32 keys of a tile, from its key 32 kb on, kv0 in the sequence, of which the
  // row sees those <= limit. (Scores and probabilities of 64 keys at once exceed
  // the registers of two waves per SIMD, and a spilled value's reload waits for
  // the copies in flight too.)
  __device__ __forceinline__ void step(uint32_t tile, int kb, int kv0, int limit, bool masked, int lane) {
    const int hl = lane / 32;
    const uint32_t kt = tile + kbase, vt = tile + vbase;
    frag_t<T> p[NM][2];
#pragma unroll
    for (int c = 0; c < NM; ++c) {
      float16_t s = zero16();
      read_ahead<SH::KS, SH::kDepth>([&](int ks) { return SH::KT::row_frag(kt, ks, c * SH::kHead + kb * 32 * SH::KT::kRowBytes); },
                                     [&](int ks, frag_t<T> f) { s = Elem<T>::mma(f, q[c][ks], s); });
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kv0 + acc_row(r, hl) > limit) s[r] = -__builtin_inff();
      }
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      top = pair_max(top) * c2;
      // The maximum moves by the row's need; one decision for the wave.
      const bool move = top > m[c] + kLazy;  // also from -inf
      if (__any(move)) {
        const float to = move ? top : m[c];
        const float alpha = m[c] == -__builtin_inff() ? 0.f : fast_exp2(m[c] - to);
        m[c] = to;
        l[c] *= alpha;
        if constexpr (STATS) e[c] *= alpha;
#pragma unroll
        for (int d = 0; d < SH::DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[c][d][r] *= alpha;
      }
      // A row that has seen no key keeps its unset maximum out of the exponent.
      const float off = m[c] == -__builtin_inff() ? 0.f : Elem<T>::kLift - m[c];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = fast_exp2(fmaf(s[r], c2, off));
        if constexpr (STATS) e[c] += s[r];
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        p[c][st] = acc_frag<T>(s, st);
        l[c] = frag_sum(p[c][st], l[c]);
      }
    }
    read_ahead<2 * SH::DB, SH::kDepth>(
        [&](int j) { return SH::VT::col_frag(vt, j % SH::DB, (kb * 32 + 16 * (j / SH::DB)) * SH::VT::kRowBytes); },
        [&](int j, frag_t<T> f) {
#pragma unroll
          for (int c = 0; c < NM; ++c) o[c][j % SH::DB] = Elem<T>::mma(f, p[c][j / SH::DB], o[c][j % SH::DB]);
        });
  }

  // Adds the state of another group's wave over the same rows and other keys,
  // which that wave has left in LDS (give).
  static constexpr int kGive = SH::DB * 4 * kWave;  // float4 per map
  static constexpr int kMl = STATS ? 3 : 2;         // numbers of a lane and map beside them
  __device__ __forceinline__ void give(float4_t* x, float* ml, int lane) {
#pragma unroll
    for (int c = 0; c < NM; ++c) {
      ml[(kMl * c) * kWave + lane] = m[c];
      ml[(kMl * c + 1) * kWave + lane] = l[c];
      if constexpr (STATS) ml[(kMl * c + 2) * kWave + lane] = e[c];
#pragma unroll
      for (int d = 0; d < SH::DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[c * kGive + (d * 4 + e) * kWave + lane] =
              float4_t{o[c][d][4 * e], o[c][d][4 * e + 1], o[c][d][4 * e + 2], o[c][d][4 * e + 3]};
    }
  }
  __device__ __forceinline__ void take(const float4_t* x, const float* ml, int lane) {
#pragma unroll
    for (int c = 0; c < NM; ++c) {
      const float m1 = ml[(kMl * c) * kWave + lane], to = fmaxf(m[c], m1);
      // An unset maximum (-inf) goes with sums that are zero, or NaN and kept.
      const float w0 = m[c] == -__builtin_inff() ? 1.f : fast_exp2(m[c] - to);
      const float w1 = m1 == -__builtin_inff() ? 1.f : fast_exp2(m1 - to);
      m[c] = to;
      l[c] = fmaf(l[c], w0, ml[(kMl * c + 1) * kWave + lane] * w1);
      if constexpr (STATS) e[c] = fmaf(e[c], w0, ml[(kMl * c + 2) * kWave + lane] * w1);
#pragma unroll
      for (int d = 0; d < SH::DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4_t y = x[c * kGive + (d * 4 + e) * kWave + lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) o[c][d][4 * e + j] = fmaf(o[c][d][4 * e + j], w0, y[j] * w1);
        }
    }
  }

  // The results of a part of the keys, whose row 0 has number `rows` of all.
  __device__ __forceinline__ void finish_part(const DiffArgs& a, int64_t rows, const DiffRow& row, int lane) {
    const int hl = lane / 32;
    const int64_t slot = rows + row.r;
#pragma unroll
    for (int c = 0; c < NM; ++c) {
      const float sum = pair_sum(l[c]), exact = STATS ? pair_sum(e[STATS ? c : 0]) : 0.f;
      if (!row.live) continue;
      float* po = a.part_o + (slot * 2 + first + c) * a.Dv;
#pragma unroll
      for (int d = 0; d < SH::DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = 32 * d + 8 * e + 4 * hl;
          if (col < a.Dv) store4t<float>(po + col, o[c][d][4 * e], o[c][d][4 * e + 1], o[c][d][4 * e + 2], o[c][d][4 * e + 3]);
        }
      if (hl == 0) {
        *reinterpret_cast<float4_t*>(a.part_ml + (slot * 2 + first + c) * 4) = float4_t{m[c], sum, exact, 0.f};
      }
    }
  }

  // The rows' results. With one map a wave, the second map's waves hand theirs
  // to the first's through `swap` (64 lanes x DB x 16 floats a pair of waves);
  // waves whose rows are not theirs to write (`mine` false) come along.
  __device__ __forceinline__ void finish(const DiffArgs& a, int b, int hk, const DiffRow& row, float4_t* swap, int lane, bool mine) {
    const int hl = lane / 32, head = hk * a.G + row.g;
    const bool in = mine && row.r < a.R;
    float* mp = STATS && a.maps != nullptr && in ? a.maps + row_at(a, b, head, row.i) * 2 * a.Dv : nullptr;
#pragma unroll
    for (int c = 0; c < NM; ++c) {
      const float sum = pair_sum(l[c]), inv = 1.f / sum;
      if constexpr (STATS) {
        const float exact = pair_sum(e[c]);
        if (a.lse != nullptr && in && hl == 0)
          a.lse[map_at(a, b, head, first + c, row.i)] = row.live ? m[c] - Elem<T>::kLift + log2f(exact) : __builtin_inff();
      }
#pragma unroll
      for (int d = 0; d < SH::DB; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int col = 32 * d + 8 * e + 4 * hl;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[c][d][4 * e + j] = row.live ? o[c][d][4 * e + j] * inv : 0.f;
          if (mp != nullptr && col < a.Dv)
            store4t<float>(mp + (first + c) * a.Dv + col, o[c][d][4 * e], o[c][d][4 * e + 1], o[c][d][4 * e + 2], o[c][d][4 * e + 3]);
        }
    }
    if constexpr (NM == 1) {
      __syncthreads();  // the key tiles, in whose place `swap` lies, have been read
      if (first == 1 && mine)
#pragma unroll
        for (int d = 0; d < SH::DB; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            swap[(d * 4 + e) * kWave + lane] = float4_t{o[0][d][4 * e], o[0][d][4 * e + 1], o[0][d][4 * e + 2], o[0][d][4 * e + 3]};
      __syncthreads();
      if (first == 1) return;
    }
    if (!in) return;
    const float lam = a.lam[head * a.lam_step];
    T* op = reinterpret_cast<T*>(a.o) + a.vo.row(b, head, row.i);
#pragma unroll
    for (int d = 0; d < SH::DB; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = 32 * d + 8 * e + 4 * hl;
        if (col >= a.Dv) continue;
        float4_t z;
        if constexpr (NM == 1) z = swap[(d * 4 + e) * kWave + lane];
        else z = float4_t{o[1][d][4 * e], o[1][d][4 * e + 1], o[1][d][4 * e + 2], o[1][d][4 * e + 3]};
        store4t<T>(op + col, fmaf(-lam, z[0], o[0][d][4 * e]), fmaf(-lam, z[1], o[0][d][4 * e + 1]),
                   fmaf(-lam, z[2], o[0][d][4 * e + 2]), fmaf(-lam, z[3], o[0][d][4 * e + 3]));
      }
  }
};

// The key tiles of one (b, key head), by WAVES waves into LDS.
template <typename T, typename SH, int HD, int WAVES>
struct KeyTiles {
  KeyCopy<T, HD, SH::BN, WAVES> k;
  KeyCopy<T, 2 * HD, SH::BN, WAVES> v;
  const T *kp, *vp;
  __device__ __forceinline__ void init(const DiffArgs& a, int b, int hk, int wave, int lane) {
    kp = reinterpret_cast<const T*>(a.k) + a.vk.row(b, 2 * hk, 0);
    vp = reinterpret_cast<const T*>(a.v) + a.vv.row(b, hk, 0);
    k.init(a.vk.ss, a.D, wave, lane);
    v.init(a.vv.ss, a.Dv, wave, lane);
  }
  // Keys kv0 .. kv0 + BN - 1; those at or past L land as zeros, whatever is there.
  __device__ __forceinline__ void issue(const DiffArgs& a, int kv0, int L, uint32_t tile, int wave) const {
#pragma unroll
    for (int c = 0; c < 2; ++c)
      k.issue(kp + c * a.vk.sh + kv0 * a.vk.ss, a.vk.ss, L - kv0, a.D, tile + c * SH::kHead, wave);
    v.issue(vp + kv0 * a.vv.ss, a.vv.ss, L - kv0, a.Dv, tile + 2 * SH::kHead, wave);
  }
};

// Maps a wave computes: accumulators of both take 4 HD registers.
template <int HD>
constexpr int kMaps = HD <= 64 ? 2 : 1;

// A workgroup's waves: row blocks times key groups times the waves that share the
// maps. Four (eight of one map), so that two workgroups share a CU where the
// registers allow it, and one's products run beside the other's exponentials:
// eight waves meeting at one barrier were 15 % slower on the long bf16 case. 128
// rows where those fill the chip, else 64 with two groups, if two tiles for each
// fit. (32 rows with four, bf16: b1 h4 s512 20.3 against 19.7 us, and twice the time
// where the keys are in parts.)
template <typename T, int HD, int BLOCKS>
struct FwdGroups {
  static constexpr int kPairs = 2 / kMaps<HD>;
  static constexpr int RB = BLOCKS, KG = 4 / RB;
  static_assert(row_blocks_fit<T, HD>(BLOCKS), "two tiles a group");
  static constexpr int WAVES = 4 * kPairs;
  static constexpr int BN = KG == 1 && HD * (int)sizeof(T) <= 256 ? 64 : 32;
};

template <typename T, int HD, int BLOCKS, bool PART, bool STATS>
__global__ __launch_bounds__((64 * FwdGroups<T, HD, BLOCKS>::WAVES), (sizeof(T) == 4 && HD == 64 ? 1 : 2)) void
diff_fwd_kernel(DiffArgs a) {
  using GR = FwdGroups<T, HD, BLOCKS>;
  constexpr int BN = GR::BN;
  using SH = FwdShape<T, HD, BN>;
  using State = FwdState<T, HD, BN, kMaps<HD>, STATS>;
  constexpr int NM = kMaps<HD>, RB = GR::RB, KG = GR::KG, ROWS = 32 * RB;
  // Two tiles a group; afterwards the groups' results, then the second map's.
  constexpr int kSums = 16 * State::kGive * RB * (KG > 1 && KG * GR::kPairs * NM / 2 > 1 ? KG * GR::kPairs * NM / 2 : 1);
  __shared__ __attribute__((aligned(1024))) unsigned char smem[KG * 2 * SH::kBytes > kSums ? KG * 2 * SH::kBytes : kSums];
  __shared__ float ml[KG > 1 ? KG / 2 * RB * GR::kPairs * NM * State::kMl * kWave : 1];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int kg = w / (RB * GR::kPairs), in_group = w % (RB * GR::kPairs), rb = in_group % RB, map = in_group / RB;
  const DiffTile t = diff_tile(a, blockIdx.x, a.n_mtiles);
  const int part = PART ? t.tile / a.n_mtiles : -1;
  const int mt = a.n_mtiles - 1 - (PART ? t.tile % a.n_mtiles : t.tile);
  const int L = diff_len(a, t.b);
  const int r0 = mt * ROWS, rw0 = r0 + 32 * rb;
  const DiffSpan all(a, r0, r0 + ROWS - 1, L), own(a, rw0, rw0 + 31, L);
  const DiffRow row(a, rw0 + lane % 32, L);
  const int n_keys = PART ? part_keys(a, L) : 0, kv_begin = PART ? part * n_keys : 0;
  const int kv_end = PART ? min(all.end, kv_begin + n_keys) : all.end;
  if (PART && kv_begin >= kv_end) return;  // not read either (live parts are counted from the rows' last key)
  const uint32_t tiles = lds_offset(smem) + kg * 2 * SH::kBytes;
  KeyTiles<T, SH, HD, RB * GR::kPairs> keys;
  keys.init(a, t.b, t.hk, in_group, lane);
  int kv0 = kv_begin + BN * kg;
  if (kv0 < kv_end) keys.issue(a, kv0, L, tiles, in_group);
  State st;
  st.init(a, t.b, t.hk, row, map, lane);
  // The workgroup goes round together, the last round maybe without a tile for every group.
  for (int first = kv_begin, cur = 0; first < kv_end; first += KG * BN, kv0 += KG * BN, cur ^= 1) {
    // The tile is there, and the group's other one has been read by its waves.
    wait_copies();
    lds_barrier();
    if (kv0 + KG * BN < kv_end) keys.issue(a, kv0 + KG * BN, L, tiles + (cur ^ 1) * SH::kBytes, in_group);
#pragma unroll
    for (int kb = 0; kb < BN / 32; ++kb) {
      const int at = kv0 + 32 * kb;
      if (at < min(own.end, kv_end)) st.step(tiles + cur * SH::kBytes, kb, at, row.limit, at + 31 > own.free, lane);
    }
  }
  // The groups' states, the upper half's joined to the lower half's.
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    float4_t* x = reinterpret_cast<float4_t*>(smem);
    const int at = (kg % half) * RB * GR::kPairs + in_group;
    __syncthreads();
    if (kg >= half && kg < 2 * half) st.give(x + at * NM * State::kGive, ml + at * NM * State::kMl * kWave, lane);
    __syncthreads();
    if (kg < half) st.take(x + at * NM * State::kGive, ml + at * NM * State::kMl * kWave, lane);
  }
  if constexpr (NM == 2) {
    if (kg != 0) return;
  }
  if constexpr (PART) {
    if (kg == 0) st.finish_part(a, ((int64_t)part * a.B * a.Hk + t.bh) * a.R, row, lane);
  } else {
    st.finish(a, t.b, t.hk, row, reinterpret_cast<float4_t*>(smem) + rb * State::kGive, lane, kg == 0);
  }
}

template <typename T, int HD>
__global__ __launch_bounds__(2 * kWave / kMaps<HD>) void diff_few_kernel(DiffArgs a) {
  constexpr int BN = 32, NM = kMaps<HD>;
  using SH = FwdShape<T, HD, BN>;
  __shared__ __attribute__((aligned(1024))) T smem[2][SH::kElems];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int mt = blockIdx.x % a.n_mtiles, hk = blockIdx.x / a.n_mtiles % a.Hk, part = blockIdx.x / a.n_mtiles / a.Hk;
  FewParts f;
  if (!f.find(a, part, lane)) return;
  const int b = __builtin_amdgcn_readfirstlane(f.b);
  const int L = diff_len(a, b);
  const DiffSpan own(a, mt * 32, mt * 32 + 31, L);
  const DiffRow row(a, mt * 32 + lane % 32, L);
  const int kv_begin = __builtin_amdgcn_readfirstlane((part - f.first) * f.keys);
  const int kv_end = min(own.end, kv_begin + __builtin_amdgcn_readfirstlane(f.keys));
  if (kv_begin >= kv_end) return;
  const uint32_t tiles = lds_offset(smem);
  KeyTiles<T, SH, HD, 2 / NM> keys;
  keys.init(a, b, hk, w, lane);
  keys.issue(a, kv_begin, L, tiles, w);
  FwdState<T, HD, BN, NM, false> st;
  st.init(a, b, hk, row, w, lane);
  int cur = 0;
  for (int kv0 = kv_begin; kv0 < kv_end; kv0 += BN, cur ^= 1) {
    wait_copies();
    lds_barrier();
    if (kv0 + BN < kv_end) keys.issue(a, kv0 + BN, L, tiles + (cur ^ 1) * SH::kBytes, w);
    st.step(tiles + cur * SH::kBytes, 0, kv0, row.limit, kv0 + BN - 1 > own.free, lane);
  }
  st.finish_part(a, ((int64_t)part * a.Hk + hk) * a.R, row, lane);
}

// Joins the parts: O_m = sum_p 2^(max_p - M) o_p / sum_p 2^(max_p - M) sum_p,
// then the difference. One row per workgroup; `lanes` threads take a part's two
// results (lanes chunks of 4 columns, the second map's after the first's), the
// workgroup's 256 / lanes sets of them every so many-th part. A row's parts are
// those up to its last key. (A wave per row, one column a lane, waited for one
// load after the other: 90 us for 256 rows of 64 parts.)
template <typename T>
__global__ __launch_bounds__(kDiffThreads) void diff_join_kernel(DiffArgs a, int lanes) {
  __shared__ float4_t sum[kDiffThreads];
  __shared__ float top[2][kDiffThreads / kWave], total[2][kDiffThreads];
  const int tid = threadIdx.x;
  const int bh = blockIdx.x / a.R, b = bh / a.Hk, hk = bh % a.Hk;
  const int L = diff_len(a, b);
  const DiffRow row(a, blockIdx.x % a.R, L);
  // The row's number in the first part, and from one part to the next.
  int64_t id = blockIdx.x, n_rows = (int64_t)a.B * a.Hk * a.R;
  int n_keys;
  if (a.few_slots + a.few_each != 0) {
    FewParts f;
    f.of(a, b, tid % kWave);
    id = ((int64_t)f.first * a.Hk + hk) * a.R + row.r;
    n_rows = (int64_t)a.Hk * a.R;
    n_keys = f.keys;
  } else {
    n_keys = part_keys(a, L);
  }
  const int np = row.live ? row.limit / n_keys + 1 : 0;
  const float4_t* ml = reinterpret_cast<const float4_t*>(a.part_ml) + id * 2;  // part p, map c: [p * n_rows * 2 + c]
  float m[2] = {-__builtin_inff(), -__builtin_inff()};
  for (int p = tid; p < np; p += kDiffThreads)
#pragma unroll
    for (int c = 0; c < 2; ++c) m[c] = fmaxf(m[c], ml[p * n_rows * 2 + c][0]);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int s = kWave / 2; s > 0; s >>= 1) m[c] = fmaxf(m[c], __shfl_xor(m[c], s));
    if (tid % kWave == 0) top[c][tid / kWave] = m[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int w = 0; w < kDiffThreads / kWave; ++w) m[c] = fmaxf(m[c], top[c][w]);

  const int chunk = tid % lanes, per_map = a.Dv / 4;
  const bool on = chunk < 2 * per_map;
  const int c = on && chunk >= per_map;
  const float* po = a.part_o + id * 2 * a.Dv + (on ? chunk : 0) * 4;
  const int64_t step = n_rows * 2 * a.Dv;
  float4_t y = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f, exact = 0.f;
#pragma unroll 4
  for (int p = tid / lanes; p < np; p += kDiffThreads / lanes) {
    const float4_t x = ml[p * n_rows * 2 + c];
    const float4_t o = *reinterpret_cast<const float4_t*>(po + p * step);
    // An unset maximum (-inf) goes with sums that are zero, or NaN and kept.
    const float w = x[0] == -__builtin_inff() ? 1.f : fast_exp2(x[0] - m[c]);
    l = fmaf(w, x[1], l);
    exact = fmaf(w, x[2], exact);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaf(w, o[j], y[j]);
  }
  sum[tid] = y;
  total[0][tid] = l;
  total[1][tid] = exact;
  __syncthreads();
  if (tid < lanes) {
    for (int s = tid + lanes; s < kDiffThreads; s += lanes) {
      y += sum[s];
      l += total[0][s];
      exact += total[1][s];
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = row.live ? y[j] * inv : 0.f;
    sum[tid] = y;
    const int head = hk * a.G + row.g;
    if (on && a.maps != nullptr) *reinterpret_cast<float4_t*>(a.maps + row_at(a, b, head, row.i) * 2 * a.Dv + chunk * 4) = y;
    if (a.lse != nullptr && (chunk == 0 || chunk == per_map))
      a.lse[map_at(a, b, head, c, row.i)] = row.live ? m[c] - Elem<T>::kLift + log2f(exact) : __builtin_inff();
  }
  __syncthreads();
  if (tid < per_map) {
    const int head = hk * a.G + row.g;
    const float lam = a.lam[head * a.lam_step];
    const float4_t z = sum[tid + per_map];
    store4t<T>(reinterpret_cast<T*>(a.o) + a.vo.row(b, head, row.i) + tid * 4, fmaf(-lam, z[0], y[0]), fmaf(-lam, z[1], y[1]),
               fmaf(-lam, z[2], y[2]), fmaf(-lam, z[3], y[3]));
  }
}

template <typename T>
int launch_join(const DiffArgs& a, hipStream_t stream) {
  int lanes = 1;
  while (lanes < a.Dv / 2) lanes *= 2;
  hipLaunchKernelGGL((diff_join_kernel<T>), dim3(uint32_t((int64_t)a.B * a.Hk * a.R)), dim3(kDiffThreads), 0, stream, a, lanes);
  return tjh::launch_status();
}

}  // namespace

namespace {
template <typename T, int HD, int BLOCKS>
int launch_fwd(DiffArgs a, hipStream_t stream) {
  using GR = FwdGroups<T, HD, BLOCKS>;
  a.n_mtiles = (a.R + 32 * GR::RB - 1) / (32 * GR::RB);
  const int64_t n = (int64_t)a.B * a.Hk * a.n_mtiles;
  // Parts are for launches that 64-row workgroups do not fill, never for 128-row ones beside them.
  if constexpr (BLOCKS != 4 || !row_blocks_fit<T, HD>(2)) {
    if (a.n_parts > 1) {
      hipLaunchKernelGGL((diff_fwd_kernel<T, HD, BLOCKS, true, true>), dim3(uint32_t(n * a.n_parts)), dim3(64 * GR::WAVES), 0,
                         stream, a);
      const int rc = tjh::launch_status();
      return rc != TJ_OK ? rc : launch_join<T>(a, stream);
    }
  }
  // Without statistics the long sweeps of 128-row workgroups save the second sum.
  if constexpr (BLOCKS == 4) {
    if (a.lse == nullptr) {
      hipLaunchKernelGGL((diff_fwd_kernel<T, HD, BLOCKS, false, false>), dim3(uint32_t(n)), dim3(64 * GR::WAVES), 0, stream, a);
      return tjh::launch_status();
    }
  }
  hipLaunchKernelGGL((diff_fwd_kernel<T, HD, BLOCKS, false, true>), dim3(uint32_t(n)), dim3(64 * GR::WAVES), 0, stream, a);
  return tjh::launch_status();
}
}  // namespace

int diff_fwd(const DiffArgs& a, int dtype, hipStream_t stream) {
  return diff_dispatch(a, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    // Four groups: fp32 d32 (bound by its products) from 128 keys on, with two / four: b1 h1 s128 12.9 / 11.8
    // us, s512 33.7 / 23.2, but s64 9.4 / 11.4.
    if constexpr (sizeof(T) == 4 && row_blocks_fit<T, HD>(1))
      if (a.Sk >= 128 && (int64_t)a.B * a.Hk * ((a.R + 63) / 64) * a.n_parts <= kCus / 2) return launch_fwd<T, HD, 1>(a, stream);
    if constexpr (row_blocks_fit<T, HD>(2))
      if (!wide_tiles(a, HD)) return launch_fwd<T, HD, 2>(a, stream);
    return launch_fwd<T, HD, 4>(a, stream);
  });
}

int diff_few_rows(const DiffArgs& args, int dtype, hipStream_t stream) {
  return diff_dispatch(args, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    DiffArgs a = args;
    constexpr int kWaves = 2 / kMaps<HD>, kLds = 2 * FwdShape<T, HD, 32>::kBytes;
    // What the LDS and the registers hold at once: two waves a SIMD at 32 dims, else one.
    constexpr int kByLds = 160 * 1024 / kLds, kByRegs = (HD == 32 ? 8 : 4) / kWaves;
    a.n_mtiles = (a.R + 31) / 32;
    const FewPlan p = few_plan(a.B, a.Hk, a.n_mtiles, a.Sk, kCus * (kByLds < kByRegs ? kByLds : kByRegs));
    a.few_slots = (int)p.slots;
    a.few_each = (int)p.each;
    a.n_parts = (int)p.total;
    hipLaunchKernelGGL((diff_few_kernel<T, HD>), dim3(uint32_t((int64_t)a.n_parts * a.Hk * a.n_mtiles)), dim3(kWave * kWaves), 0,
                       stream, a);
    const int rc = tjh::launch_status();
    return rc != TJ_OK ? rc : launch_join<T>(a, stream);
  });
}

}  // namespace tj
