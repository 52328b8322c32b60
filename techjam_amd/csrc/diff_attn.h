// Differential attention for gfx950: shared by its forward, backward and
// cached kernels (diff_attn_fwd.hip, diff_attn_bwd_kv.hip, diff_attn_bwd_q.hip,
// diff_attn.hip).
//
// Head h of H is the difference of two softmax maps over one value head,
//
//   O_h = (P_0 - lam_h P_1) V,   P_m = softmax(scale Q_{2h+m} K_{2h'+m}^T),
//
// with h' = h / G the key head that G = H / Hk query heads share. The G heads
// of one key head are handled together: their query rows are numbered
// r = i G + g (token i, head g of the group), so that neighbouring rows see
// nearly the same keys, one sweep over K and V serves the whole group, and the
// sums over the group in dK and dV are sums over rows.
#pragma once

#include "attn_tiles.h"

namespace tj {

struct DiffArgs {
  const void *q, *k, *v;
  void* o;
  float* maps;             // [B, H, Sq, 2, Dv] P_0 V and P_1 V for the backward pass, or null
  View4 vq, vk, vv, vo;
  int B, H, Hk, G, D, Dv;
  int Sq, Sk;              // query tokens, key tokens (capacity of a cache)
  int R;                   // rows of one key head: Sq * G
  float scale;
  int causal;
  int cached;              // token i stands at position len - Sq + i instead of i
  const float* lam;
  int lam_step;            // elements between the weights of two heads: 0 or 1
  const int32_t* len;      // [B] or null
  float* lse;              // [B, H, 2, Sq] log2 of a row's sum of 2^(score log2 e), +inf for empty rows; or null
  int n_mtiles;
  // Key parts: n_parts of every sequence (part_keys), which leave unnormalised sums
  // [n_parts, B, Hk, R, 2, Dv] and (maximum, sum, sum before rounding, -) [n_parts, B, Hk, R, 2, 4];
  // or, for few rows, as many of each sequence as its length asks for (FewParts),
  // n_parts in all, [n_parts, Hk, R, ...]. part_o null: sweeps run whole.
  int n_parts, few_slots, few_each;
  float *part_o, *part_ml;
  // Backward.
  const void* dout;
  View4 vdo, vdq, vdk, vdv;
  void *dq, *dk, *dv;
  float* dlam;             // [H], or [1] when lam_step is 0
  int n_lam;
  float* delta;            // [B, H, 2, Sq] rowsum(dO o O_m)
  float* gsum;             // [B, H, Sq] rowsum(P_1 o dP), the row's part of -dlam
  float* stat;             // [B, H, stat_rows(Sq) / 32, 4, 32] what the dK, dV kernel reads of a row
  float* peak;             // [B, Hk, 2, kPeakParts] largest norms of dO and V rows (fp16 operands)
  int n_peaks;
};

constexpr int kPeakParts = 64;
constexpr int kDiffThreads = 256;

// Keys of sequence b, clipped to what is there; the same in every lane.
__device__ __forceinline__ int diff_len(const DiffArgs& a, int b) {
  const int n = a.len == nullptr ? a.Sk : min(a.Sk, max(0, a.len[b]));
  return __builtin_amdgcn_readfirstlane(n);
}

// Keys of one of n_parts parts of a sequence of L: they share the sequence, not
// the capacity, so that a short sequence in a long cache is swept by as many.
constexpr int kPartKeys = 512;
__device__ __forceinline__ int part_keys(const DiffArgs& a, int L) {
  return max(kPartKeys, ((L + a.n_parts - 1) / a.n_parts + 63) / 64 * 64);
}

// Products with fp16 operands: powers of two that bring the largest possible |dS|,
// 2 |dO_i| |V_j| max(1, |lam|), near 2^15, so that small gradients and small
// probabilities keep fp16's bits. dQ is a sum over keys, so there every row has
// its own, by its dO (of) and the largest V row: a row's bits do not depend on
// how large the gradients of others are.
// dK sums over rows and has one for all of a (b, key head), by the largest dO
// row: dS of a row r times smaller keeps 11 bits down to P of about 2^-26 r, and
// what lies below is off by at most 2^-37 of the largest possible |dS|. 1 for the
// other types.
template <typename T>
struct DsLift {
  float o = 1.f, v = 1.f;  // the largest norms of dO and V rows
  int ew = 0;              // exponent of the heads' largest max(1, |lam|)
  __device__ __forceinline__ DsLift(const DiffArgs& a, int bh, int hk, int lane) {
    if constexpr (std::is_same<T, half_t>::value) {
      const float* pk = a.peak + (int64_t)bh * 2 * kPeakParts;
      o = lane < a.n_peaks ? pk[lane] : 0.f;
      v = lane < a.n_peaks ? pk[kPeakParts + lane] : 0.f;
#pragma unroll
      for (int m = 32; m > 0; m >>= 1) {
        o = fmaxf(o, __shfl_xor(o, m));
        v = fmaxf(v, __shfl_xor(v, m));
      }
      float w = 1.f;
      for (int g = 0; g < a.G; ++g) {
        const float l = fabsf(a.lam[(hk * a.G + g) * a.lam_step]);
        if (l < 3e38f) w = fmaxf(w, l);
      }
      frexpf(w, &ew);
    }
  }
  // For rows whose dO has at most this norm.
  __device__ __forceinline__ float of(float norm) const {
    if constexpr (!std::is_same<T, half_t>::value) return 1.f;
    // Exponents rather than products: the norms' product may leave fp32.
    int ex, ey;
    frexpf(norm, &ex);
    frexpf(v, &ey);
    if (!(norm > 0.f) || !(norm < 3e38f) || !(v > 0.f)) return 1.f;  // a row that is not finite is lost anyway
    return ldexpf(1.f, min(max(14 - ex - ey - ew, -100), 100));
  }
  __device__ __forceinline__ float all() const { return of(o); }
};

// A row's place in the arrays [B, H, Sq].
__device__ __forceinline__ int64_t row_at(const DiffArgs& a, int b, int head, int i) {
  return ((int64_t)b * a.H + head) * a.Sq + i;
}
// Its place in the arrays [B, H, 2, Sq], for map c.
__device__ __forceinline__ int64_t map_at(const DiffArgs& a, int b, int head, int c, int i) {
  return (((int64_t)b * a.H + head) * 2 + c) * a.Sq + i;
}

// A row's numbers in `stat`: log2 of P_0's and P_1's factor (minus lse, plus the
// lift), -delta_0 and lam delta_1 (lifted). Rows that are not there, up to the
// next multiple of 32, have -inf, -inf, 0, 0: P is 0.
__host__ __device__ __forceinline__ int64_t stat_rows(int64_t S) { return (S + 31) / 32 * 32; }
__device__ __forceinline__ float* stat_at(const DiffArgs& a, int b, int head, int i, int which) {
  return a.stat + (((int64_t)b * a.H + head) * stat_rows(a.Sq) + i / 32 * 32) * 4 + which * 32 + i % 32;
}

// The same for P_0 - lam P_1 (at most 1 + |lam|).
template <typename T>
__device__ __forceinline__ float p_lift(const DiffArgs& a, int hk) {
  if constexpr (!std::is_same<T, half_t>::value) {
    return 1.f;
  } else {
    float lam_max = 0.f;
    for (int g = 0; g < a.G; ++g) {
      const float l = fabsf(a.lam[(hk * a.G + g) * a.lam_step]);
      if (l < 3e38f) lam_max = fmaxf(lam_max, l);
    }
    int e;
    frexpf(1.f + lam_max, &e);
    return ldexpf(1.f, min(max(15 - e, -100), 14));
  }
}

// A workgroup's tile and (b, key head). Consecutive ids run on the XCDs in
// turn, so the (b, key head) index varies fastest: with a multiple of eight of
// them the tiles that share K and V also share an XCD's L2. Tiles with the
// most keys come first.
struct DiffTile {
  int b, hk, bh, tile;
};
__device__ __forceinline__ DiffTile diff_tile(const DiffArgs& a, int id, int tiles) {
  const int bhn = a.B * a.Hk;
  DiffTile t;
  t.bh = id % bhn;
  t.tile = id / bhn;
  t.b = t.bh / a.Hk;
  t.hk = t.bh % a.Hk;
  return t;
}

// Whether there are 128-row tiles enough for workgroups to take them rather than 64-row ones:
// two rounds of them where two fit a CU; where one does, one, and two of causal ones,
// whose lengths differ. us with 128 / 64 rows, bf16, 4096 tokens. 64 dims, causal: forward
// with sums 512 tiles 164 / 156, 640 tiles 175 / 186, 768 tiles 201 / 212, 1024 tiles 245 / 263, dQ
// 172 / 146, 178 / 174, 196 / 199, 257 / 255; not causal, forward 226 / 247, 333 / 309, 343 / 365,
// 437 / 481, dQ 233 / 246, 344 / 309, 354 / 366, 455 / 484. So 1024 is where both gain whatever the
// mask; the causal forward alone would from 640 on. 32 dims, causal forward: 512 tiles 107 / 90, 768
// tiles 130 / 123, 1024 tiles 154 / 161. 128 dims forward, 290 tiles 68 / 81, causal 256 tiles
// 174 / 141, 512 tiles 227 / 280.
inline bool wide_tiles(const DiffArgs& a, int hd) {
  return (int64_t)a.B * a.Hk * ((a.R + 127) / 128) >= (hd == 128 ? (a.causal ? 512 : 256) : 1024);
}

// Workgroups of four waves have `blocks` blocks of 32 rows (4, 2 or 1) times 4 / blocks
// groups of key tiles. Whether two tiles for each of those groups fit the LDS.
template <typename T, int HD>
constexpr bool row_blocks_fit(int blocks) { return 4 / blocks * HD * (int)sizeof(T) <= 512; }

int diff_fwd(const DiffArgs& a, int dtype, hipStream_t stream);
int diff_few_rows(const DiffArgs& a, int dtype, hipStream_t stream);
int diff_bwd_kv(const DiffArgs& a, int dtype, hipStream_t stream);
int diff_bwd_q(const DiffArgs& a, int dtype, hipStream_t stream);

// f.operator()<T, HD, DVP>() for the smallest instance that holds D and Dv:
// head dims up to 32, 64 or 128 with values up to twice as wide.
template <typename F>
int diff_dispatch(const DiffArgs& a, int dtype, F&& f) {
  const int need = a.D > (a.Dv + 1) / 2 ? a.D : (a.Dv + 1) / 2;
  auto by_dim = [&](auto t) {
    using T = decltype(t);
    if (need <= 32) return f(t, std::integral_constant<int, 32>{});
    if (need <= 64) return f(t, std::integral_constant<int, 64>{});
    return f(t, std::integral_constant<int, 128>{});
  };
  if (dtype == TJ_F32) return by_dim(float{});
  if (dtype == TJ_F16) return by_dim(half_t{});
  return by_dim(bf16_t{});
}

}  // namespace tj
