// Softmax attention with grouped heads for gfx950: shared by the kernels of
// packed sequences (packed_attn_fwd.hip, packed_attn_bwd.hip), of drafted tokens
// against a cache (tree_attn.hip) and their entry points (grouped_attn.hip).
//
//   O_h = softmax(scale Q_h K_{h'}^T) V_{h'},   h' = h / G,  G = H / Hk.
//
// The G query heads of one key head are handled together: their query rows are
// numbered r = i G + g (token i, head g of the group), so that neighbouring rows
// see nearly the same keys, one sweep over K and V serves the whole group, and
// the sums over the group in dK and dV are sums over rows.
#pragma once

#include "attn_tiles.h"

namespace tj {

// Strided [rows, heads, dim] view with unit dim stride, the others below 2^31.
struct View3 {
  int64_t st, sh;
  __device__ __forceinline__ int64_t row(int64_t t, int h) const { return t * st + h * sh; }
};

// Division of row numbers (below 2^31) by the group's size, by a product: with 2^shift >= n > 2^(shift - 1)
// and mul = ceil(2^(31 + shift) / n), x mul / 2^(31 + shift) is off by less than x / 2^31 / n.
struct Divisor {
  uint32_t mul;
  int shift, n;
  static Divisor of(int n) {
    int shift = 0;
    while ((int64_t(1) << shift) < n) ++shift;
    return Divisor{uint32_t(((uint64_t(1) << (31 + shift)) + n - 1) / n), shift, n};
  }
};
__device__ __forceinline__ int operator/(int x, Divisor d) { return (int)(__umulhi((uint32_t)x * 2, d.mul) >> d.shift); }
__device__ __forceinline__ int operator%(int x, Divisor d) { return x - x / d * d.n; }

struct PackedArgs {
  const void *q, *k, *v;
  void* o;
  View3 vq, vk, vv, vo;
  int T, N;                // tokens in all, sequences
  int H, Hk, G, D, Dv;
  Divisor by_group;        // G
  float scale;
  int causal;
  const int32_t* off;      // [N + 1]
  const int32_t* len;      // [N] valid tokens of each sequence's rows, or null: all
  float* lse;              // [T, H] log2 of a row's sum of 2^(score log2 e); or null
  void* rest;              // kRestLift times what rounding took from o, in o's type and layout (16-bit types); or null
  int n_slots;             // of the launch, see Region
  // Backward.
  const void *out, *dout;
  View3 vdo, vdq, vdk, vdv;
  void *dq, *dk, *dv;
  float* stat;             // [slots of 32 tokens, H, 2, 32] what the dK, dV kernel reads of a row
  float* peak;             // [slots of 64 tokens, Hk, 2] largest norms of dO and V rows (fp16 operands)
  int shares;              // workgroups that share the rows of a key tile
  float* part;             // [shares, T, Hk, Dv + D] their sums for dV and dK; used where there are several
};

// The rows fall into regions: what lies before the first sequence, the sequences,
// and what lies behind the last, whose rows are written as zeros. Region j of
// regions() starts at token edge(j).
//
// Where a tile of `unit` rows belongs is found without a list of tiles, which would
// cost a launch, and without the lengths on the host, which would cost a wait: region
// j's tiles have the slots from slot(j) = edge(j) per / unit + j on, rows counted
// `per` a token. A region of n rows has at most slot(j + 1) - slot(j) tiles, so the
// slots do not overlap, and at most one a region is left over. Offsets
// are clipped to 0 .. T, and offsets out of order give wrong rows, but none outside.
struct Region {
  int index, start, rows, len, tile;

  __device__ __forceinline__ static int regions(const PackedArgs& a) { return a.N + 2; }
  __device__ __forceinline__ static int edge(const PackedArgs& a, int j) {
    if (j <= 0) return 0;
    return j > a.N + 1 ? a.T : min(a.T, max(0, a.off[j - 1]));
  }
  __device__ __forceinline__ static int slot(int edge, int j, int per, int unit) { return (int)((int64_t)edge * per / unit) + j; }
  // Tokens among the first rows of region j.
  __device__ __forceinline__ static int tokens(const PackedArgs& a, int j, int rows) {
    if (j <= 0 || j > a.N) return 0;
    return a.len == nullptr ? rows : min(rows, max(0, a.len[j - 1]));
  }

  // The region and tile of slot `at`, in every lane of the wave that asks; false for a slot left
  // over. Sixty-four regions are looked at at a time.
  __device__ __forceinline__ bool find(const PackedArgs& a, int at, int per, int unit, int lane) {
    int lo = 0, n = regions(a);
    while (n > 1) {
      const int step = (n + kWave - 1) / kWave, j = lo + lane * step;
      const bool in = lane * step < n;
      const int s = in ? slot(edge(a, j), j, per, unit) : 0;
      const int before = max(1, (int)__popcll(__ballot(in && s <= at)));
      lo += (before - 1) * step;
      n = min(step, n - (before - 1) * step);
    }
    index = __builtin_amdgcn_readfirstlane(lo);
    start = __builtin_amdgcn_readfirstlane(edge(a, index));
    rows = max(0, __builtin_amdgcn_readfirstlane(edge(a, index + 1)) - start);
    len = __builtin_amdgcn_readfirstlane(tokens(a, index, rows));
    tile = at - slot(start, index, per, unit);
    return there(per, unit);
  }
  // Offsets out of order may have led anywhere.
  __device__ __forceinline__ bool there(int per, int unit) const {
    return tile >= 0 && (int64_t)tile * unit < (int64_t)rows * per;
  }

  // Sums and maxima of non-negative numbers over a wave, by DPP: a shuffle through the LDS takes
  // five times as long.
  template <typename Op>
  __device__ __forceinline__ static int over_wave(int x, Op&& op) {
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // row_shr:1, 2, 4, 8
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // row_bcast:15, 31
    x = op(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, kWave - 1);
  }

  // The at-th tile of all when those that take longest come first, so that no long one is left
  // for the end: a causal sequence of n tiles has one of each length from 1 to n (the
  // last the longest, or with `down` the first), another n of length n. Tiles without tokens
  // come last. One wave counts, by halving the range of lengths: half a microsecond, where a
  // launch that sorts would take several. For up to kRanked regions.
  static constexpr int kChunks = 4, kRanked = kChunks * kWave;
  __device__ __forceinline__ bool ranked(const PackedArgs& a, int at, int per, int unit, bool down, int lane) {
    int n[kChunks], from_[kChunks], rows_[kChunks], len_[kChunks], count = 0, top = 0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int j = c * kWave + lane;
      n[c] = from_[c] = rows_[c] = len_[c] = 0;
      if (c * kWave < regions(a) && j < regions(a)) {
        from_[c] = edge(a, j);
        rows_[c] = max(0, edge(a, j + 1) - from_[c]);
        len_[c] = tokens(a, j, rows_[c]);
        n[c] = (len_[c] * per + unit - 1) / unit;
      }
      count += n[c];
      top = max(top, n[c]);
    }
    auto sum = [](int x, int y) { return x + y; };
    count = over_wave(count, sum);
    const bool live = at < count;
    int lo = 0, rank;
    if (live) {
      int hi = over_wave(top, [](int x, int y) { return max(x, y); }), beyond = 0;  // more than `at` tiles are longer than lo, `beyond` <= at than hi
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        int x = 0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          if (c * kWave < regions(a)) x += a.causal ? max(0, n[c] - mid) : (n[c] > mid ? n[c] : 0);
        x = over_wave(x, sum);
        if (x > at) lo = mid;
        else {
          hi = mid;
          beyond = x;
        }
      }
      rank = at - beyond;
    } else {
      rank = at - count;
    }
    // Which region: among those with a tile of this length the rank-th, or the rank-th of the tiles without tokens.
    tile = a.causal ? lo : (live ? rank % (lo + 1) : 0);
    if (live && !a.causal) rank /= lo + 1;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (c * kWave >= regions(a)) break;
      uint64_t who;
      if (live) {
        const bool has = a.causal ? n[c] > lo : n[c] == lo + 1;
        const uint64_t mask = __ballot(has);
        const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        who = __ballot(has && before == rank);
        rank -= (int)__popcll(mask);
      } else {
        int upto = (rows_[c] * per + unit - 1) / unit - n[c];
        const int own = upto;
#pragma unroll
        for (int s = 1; s < kWave; s <<= 1) {
          const int x = __shfl_up(upto, s);
          if (lane >= s) upto += x;
        }
        who = __ballot(rank < upto && rank >= upto - own);
        if (who != 0) tile = rank - __builtin_amdgcn_readlane(upto - own, __builtin_ctzll(who));
        else rank -= __builtin_amdgcn_readlane(upto, kWave - 1);
      }
      if (who != 0) {
        const int at = __builtin_ctzll(who), tiles = __builtin_amdgcn_readlane(n[c], at);
        index = c * kWave + at;
        if (!live) tile += tiles;
        else if (a.causal && down) tile = tiles - 1 - tile;
        start = __builtin_amdgcn_readlane(from_[c], at);
        rows = __builtin_amdgcn_readlane(rows_[c], at);
        len = __builtin_amdgcn_readlane(len_[c], at);
        return there(per, unit);
      }
    }
    return false;
  }

  // The tile of workgroup `at`, of as many slots as the launch has, for all of its waves: the first one looks, as the
  // others would take the vector unit's time for the same numbers. `told`: six integers of LDS.
  __device__ __forceinline__ bool take(const PackedArgs& a, int at, int per, int unit, bool down, int tid, int* told) {
    const int lane = tid % kWave;
    if (tid < kWave) {
      const bool any = regions(a) <= kRanked ? ranked(a, at, per, unit, down, lane)
                                             : find(a, down ? at : a.n_slots - 1 - at, per, unit, lane);
      if (lane == 0) {
        told[0] = any;
        told[1] = index;
        told[2] = start;
        told[3] = rows;
        told[4] = len;
        told[5] = tile;
      }
    }
    __syncthreads();
    index = __builtin_amdgcn_readfirstlane(told[1]);
    start = __builtin_amdgcn_readfirstlane(told[2]);
    rows = __builtin_amdgcn_readfirstlane(told[3]);
    len = __builtin_amdgcn_readfirstlane(told[4]);
    tile = __builtin_amdgcn_readfirstlane(told[5]);
    return __builtin_amdgcn_readfirstlane(told[0]) != 0;
  }
};

inline int64_t region_slots(int64_t T, int64_t N, int64_t per, int64_t unit) { return T * per / unit + N + 2; }

struct TreeArgs {
  const void *q, *k, *v;
  void* o;
  View4 vq, vk, vv, vo;
  int B, H, Hk, G, D, Dv;
  int Sq, Sk;              // drafted tokens, capacity of the cache
  int R;                   // rows of one key head: Sq * G
  Divisor by_group;        // G
  float scale;
  const int32_t* len;      // [B]
  const int32_t* parents;  // [B, Sq], or null: a chain
  int n_mtiles;
  // Parts of the keys (FewParts), n_parts in all, which leave unnormalised sums [n_parts, Hk, R, Dv] and
  // (maximum, sum, whether the row is there, -) [n_parts, Hk, R, 4]. part_o null: sweeps run whole.
  int n_parts, few_slots, few_each;
  float *part_o, *part_ml;
  int32_t* plan;           // [B, 2] a sequence's first part, the keys of each
};

// What rounding took from the output (PackedArgs::rest) is kept times this. fp16: 2^11, as the rest is 2^-11 of the output
// and would lose its bits below 2^-24 where the output is small; with it the two are off by 2^-22 of the output, and by
// 2^-36 at the most below 2^-14. The largest, 16 of 65504, becomes 2^15. bf16 has fp32's exponents.
template <typename T>
constexpr float kRestLift = std::is_same<T, half_t>::value ? 2048.f : 1.f;

constexpr float kLazy = 8.f;  // the running maximum moves when a row's maximum grows by more than 2^8

// HD: head dim computed, 32, 64, 96 or 128; a row of an LDS tile holds the next power of two.
template <typename T, int HD, int BNT>
struct SweepShape {
  static constexpr int W = HD <= 32 ? 32 : (HD <= 64 ? 64 : 128);
  static constexpr int BN = BNT;       // keys of a tile
  using Rows = LdsRows<T, W>;
  static constexpr int KS = HD / 16;   // k-steps over the head dim
  static constexpr int DB = HD / 32;   // output blocks
  static constexpr int kDepth = sizeof(T) == 2 && HD > 32 ? 2 : 0;
  static constexpr int kTensor = BN * W * (int)sizeof(T), kBytes = 2 * kTensor;  // K's tile, then V's
};

// A lane's row of the tile's (region or sequence, key head): its token, head, and
// the last key it sees.
struct SweepRow {
  int i, g, limit;
  bool live;
};

// The 32 rows of a wave between memory and registers, through an LDS tile of its own. A fragment
// holds a row's elements lane by lane, so that one instruction would touch 32 rows, 32 or
// 16 bytes of each; through the tile it moves whole rows.
template <typename T, int HD>
struct WaveRows {
  using SH = SweepShape<T, HD, 32>;
  using Rows = typename SH::Rows;
  static constexpr int kBytes = 32 * Rows::kRowBytes;
  static constexpr int kPer = kWave / Rows::kChunks, N = 32 / kPer;  // rows of an instruction, instructions
  typedef T vec_t __attribute__((ext_vector_type(Rows::kVec)));
  template <typename V>
  __device__ __forceinline__ static void put(uint32_t at, V x) { *(__attribute__((address_space(3))) V*)(uintptr_t)at = x; }

  // The tokens and heads of the rows that the lane moves, from row `first` of the (region or sequence, key head)
  // on: tokens from that of row `first`, heads from the group's first. Counted up rather than divided.
  struct Places {
    int row, i[N], g[N];
    __device__ __forceinline__ Places(int first, Divisor group, int lane) : row(first + lane / Rows::kChunks) {
      const int q = kPer / group, rest = kPer - q * group.n, token = first / group;
      int at = row / group, head = row - at * group.n;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        i[n] = at - token;
        g[n] = head;
        at += q;
        head += rest;
        if (head >= group.n) {
          head -= group.n;
          ++at;
        }
      }
    }
    __device__ __forceinline__ int64_t offset(int n, int st, int sh) const { return (int64_t)i[n] * st + (int64_t)g[n] * sh; }
    __device__ __forceinline__ bool before(int n, int end) const { return row + n * kPer < end; }
  };

  // The lane's chunks of the rows before `end`; p: the first row's token and the group's first head, whose
  // tokens are st and heads sh elements apart.
  __device__ __forceinline__ static void read(vec_t x[N], const T* p, int64_t st, int64_t sh, int width, const Places& places,
                                              int end, int lane) {
    const int col = lane % Rows::kChunks * Rows::kVec;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < Rows::kVec; ++j) x[n][j] = (T)0.f;
      if (places.before(n, end) && col < width)
        x[n] = *reinterpret_cast<const vec_t*>(p + col + places.offset(n, (int)st, (int)sh));
    }
  }
  // They, as the wave's fragments.
  __device__ __forceinline__ static void turn(const vec_t x[N], uint32_t tile, int lane, frag_t<T> f[SH::KS]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = n * kPer + lane / Rows::kChunks;
      put(tile + r * Rows::kRowBytes + (((lane % Rows::kChunks) ^ Rows::swizzle(r)) << 4), x[n]);
    }
    wait_lds();
    const uint32_t base = tile + Rows::lane_row(lane);
#pragma unroll
    for (int ks = 0; ks < SH::KS; ++ks) f[ks] = Rows::row_frag(base, ks, 0);
  }

  // Accumulators of a transposed product to rows of memory: value(d, c): the four values of the lane's row from
  // column 32 d + 8 c + 4 (lane / 32) on.
  template <typename V>
  __device__ __forceinline__ static void write(T* p, int64_t st, int64_t sh, int width, const Places& places, int end,
                                               uint32_t tile, int lane, V&& value) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    const int r = lane % 32;
#pragma unroll
    for (int d = 0; d < SH::DB; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4_t y = value(d, c);
        const int col = 32 * d + 8 * c + 4 * (lane / 32);
        put(tile + r * Rows::kRowBytes + (((col / Rows::kVec) ^ Rows::swizzle(r)) << 4) + (col % Rows::kVec) * (int)sizeof(T),
            t4{(T)y[0], (T)y[1], (T)y[2], (T)y[3]});
      }
    wait_lds();
    const int col = lane % Rows::kChunks * Rows::kVec;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = n * kPer + lane / Rows::kChunks;
      const vec_t x = lds_at<vec_t>(tile + r * Rows::kRowBytes + (((lane % Rows::kChunks) ^ Rows::swizzle(r)) << 4));
      if (places.before(n, end) && col < width) *reinterpret_cast<vec_t*>(p + col + places.offset(n, (int)st, (int)sh)) = x;
    }
  }
};

// The running state of a wave's 32 rows. Scores are formed transposed, S^T = K Q^T,
// so that a lane holds scores of ONE row: maximum and sum are per lane (the other
// half of the wave holds the other keys), and the probabilities turn into the B
// operand of O^T = V^T P^T where they stand. (Two blocks of 32 rows a wave read every fragment from LDS
// half as often, but leave a SIMD one wave of 400 registers, whose products and exponentials take turns:
// 1310 us instead of 857 for two sequences of 1904 and 14480 tokens, 16 heads on 8, 128 dims, bf16.)
//
// The output is divided by the sum of the probabilities as they were rounded for its
// product (to the inputs' type: fp32 MFMAs would take 16 times as long): a dominant
// key's rounding cancels, and two go into one instruction. What the backward pass
// gets (STATS) is the sum of the unrounded ones, so that its P sums to 1 as exactly
// as fp32 does.
template <typename T, int HD, int BN, bool STATS>
struct SweepState {
  using SH = SweepShape<T, HD, BN>;
  frag_t<T> q[SH::KS];
  float16_t o[SH::DB];
  float m, l;          // maximum in log2 units, the lane's part of the sum
  float e;             // of the unrounded ones
  float c2;            // |scale| log2 e
  uint32_t kbase, vbase;  // the lane's places in a tile

  // With q's rows as they are in memory.
  __device__ __forceinline__ void init(float scale, int lane) {
    kbase = SH::Rows::lane_row(lane);
    vbase = SH::Rows::lane_col(lane) + SH::kTensor;
    // A negative scale turns q's sign, so that the largest score is the largest
    // product; a zero one becomes too small to matter, so that masked stays -inf.
    c2 = fmaxf(fabsf(scale) * kLog2e, 1e-37f);
    if (scale < 0.f)
#pragma unroll
      for (int ks = 0; ks < SH::KS; ++ks)
#pragma unroll
        for (int j = 0; j < 8; ++j) q[ks][j] = -q[ks][j];
    m = -__builtin_inff();
    l = e = 0.f;
#pragma unroll
    for (int d = 0; d < SH::DB; ++d) o[d] = zero16();
  }

  // 32 keys of a tile, from its key 32 kb on. mask(s): sets the scores of keys that the lane's
  // row does not see to -inf.
  template <typename Mask>
  __device__ __forceinline__ void step(uint32_t tile, int kb, Mask&& mask) {
    const uint32_t kt = tile + kbase, vt = tile + vbase;
    float16_t s = zero16();
    read_ahead<SH::KS, SH::kDepth>([&](int ks) { return SH::Rows::row_frag(kt, ks, kb * 32 * SH::Rows::kRowBytes); },
                                   [&](int ks, frag_t<T> f) { s = Elem<T>::mma(f, q[ks], s); });
    mask(s);
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
    top = pair_max(top) * c2;
    // The maximum moves by the row's need; one decision for the wave.
    const bool move = top > m + kLazy;  // also from -inf
    if (__any(move)) {
      const float to = move ? top : m;
      const float alpha = m == -__builtin_inff() ? 0.f : fast_exp2(m - to);
      m = to;
      l *= alpha;
      if constexpr (STATS) e *= alpha;
#pragma unroll
      for (int d = 0; d < SH::DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    // A row that has seen no key keeps its unset maximum out of the exponent.
    const float off = m == -__builtin_inff() ? 0.f : Elem<T>::kLift - m;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(fmaf(s[r], c2, off));
      if constexpr (STATS) e += s[r];
    }
    frag_t<T> p[2];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      p[st] = acc_frag<T>(s, st);
      l = frag_sum(p[st], l);
    }
    read_ahead<2 * SH::DB, SH::kDepth>(
        [&](int j) { return SH::Rows::col_frag(vt, j % SH::DB, (kb * 32 + 16 * (j / SH::DB)) * SH::Rows::kRowBytes); },
        [&](int j, frag_t<T> f) { o[j % SH::DB] = Elem<T>::mma(f, p[j / SH::DB], o[j % SH::DB]); });
  }

  // Adds the state of another wave over the same rows and other keys, which that wave has left
  // in LDS (give).
  static constexpr int kGive = SH::DB * 4 * kWave;  // float4
  static constexpr int kMl = STATS ? 3 : 2;         // numbers of a lane beside them
  __device__ __forceinline__ void give(float4_t* x, float* ml, int lane) {
    ml[lane] = m;
    ml[kWave + lane] = l;
    if constexpr (STATS) ml[2 * kWave + lane] = e;
#pragma unroll
    for (int d = 0; d < SH::DB; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) x[(d * 4 + c) * kWave + lane] = four(d, c);
  }
  __device__ __forceinline__ void take(const float4_t* x, const float* ml, int lane) {
    const float m1 = ml[lane], to = fmaxf(m, m1);
    // An unset maximum (-inf) goes with sums that are zero, or NaN and kept.
    const float w0 = m == -__builtin_inff() ? 1.f : fast_exp2(m - to);
    const float w1 = m1 == -__builtin_inff() ? 1.f : fast_exp2(m1 - to);
    m = to;
    l = fmaf(l, w0, ml[kWave + lane] * w1);
    if constexpr (STATS) e = fmaf(e, w0, ml[2 * kWave + lane] * w1);
#pragma unroll
    for (int d = 0; d < SH::DB; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4_t y = x[(d * 4 + c) * kWave + lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][4 * c + j] = fmaf(o[d][4 * c + j], w0, y[j] * w1);
      }
  }

  // The lane's four values from column 32 d + 8 c + 4 (lane / 32) on.
  __device__ __forceinline__ float4_t four(int d, int c) const {
    return float4_t{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
  }
};

// The key tiles of one key head, by WAVES waves into LDS.
template <typename T, typename SH, int WAVES>
struct SweepTiles {
  using Copy = KeyCopy<T, SH::W, SH::BN, WAVES>;
  Copy k, v;
  const T *kp, *vp;
  int64_t ks, vs;
  int D, Dv;
  // k0, v0: the first key; rows `ks_`, `vs_` elements apart.
  __device__ __forceinline__ void init(const T* k0, const T* v0, int64_t ks_, int64_t vs_, int d, int dv, int wave, int lane) {
    kp = k0;
    vp = v0;
    ks = ks_;
    vs = vs_;
    D = d;
    Dv = dv;
    k.init(ks, D, wave, lane);
    v.init(vs, Dv, wave, lane);
  }
  // Keys kv0 .. kv0 + BN - 1; those at or past `end` land as zeros, whatever is there.
  __device__ __forceinline__ void issue(int kv0, int end, uint32_t tile, int wave) const {
    k.issue(kp + kv0 * ks, ks, end - kv0, D, tile, wave);
    v.issue(vp + kv0 * vs, vs, end - kv0, Dv, tile + SH::kTensor, wave);
  }
};

// f(T{}, integral_constant<HD>) for the smallest instance that holds D and Dv.
template <typename F>
int grouped_dispatch(int D, int Dv, int dtype, F&& f) {
  const int need = D > Dv ? D : Dv;
  auto by_dim = [&](auto t) {
    if (need <= 32) return f(t, std::integral_constant<int, 32>{});
    if (need <= 64) return f(t, std::integral_constant<int, 64>{});
    if (need <= 96) return f(t, std::integral_constant<int, 96>{});
    return f(t, std::integral_constant<int, 128>{});
  };
  if (dtype == TJ_F32) return by_dim(float{});
  if (dtype == TJ_F16) return by_dim(half_t{});
  return by_dim(bf16_t{});
}

// How a call on drafted tokens runs: workgroups of `blocks` blocks of 32 rows, and the parts of the keys.
struct TreePlan {
  int blocks;
  FewPlan parts;
  bool whole() const { return parts.each == 1; }
};
TreePlan tree_plan(const TreeArgs& a, int dtype);
int tree_fwd(const TreeArgs& a, const TreePlan& p, int dtype, hipStream_t stream);

// Whether sequences of ordinary length are causal and long, so that tiles of one launch take very different times.
inline bool long_triangles(const PackedArgs& a) { return a.causal && a.T / (a.N > 0 ? a.N : 1) >= 2048; }

int packed_fwd(const PackedArgs& a, int dtype, hipStream_t stream);
int packed_bwd_shares(int dtype, int64_t T, int64_t N, int64_t H, int64_t Hk);
int packed_bwd(const PackedArgs& a, int dtype, hipStream_t stream);

}  // namespace tj
