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
//
// Element types: fp16 and bf16 run 32x32x16 MFMAs, fp32 runs 32x32x2 fp32
// MFMAs (1/16 of the rate; nothing is rounded to fewer bits). The three share
// every kernel: an operand fragment is 8 consecutive k of one row or column
// per lane, and fp32 contracts it with eight MFMAs, one k of each lane half
// at a time, which only reorders the sum.
#pragma once

#include "tj_common.h"

typedef __bf16 bf16_t;
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

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
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kDiffBufferFlags = 0x00020000;  // raw buffer resource word 3 on gfx950

template <typename T>
struct Elem;

template <>
struct Elem<half_t> {
  typedef half8_t frag;
  static constexpr bool kWide = false;
  // 2^6: unnormalised probabilities reach 2^(6+8) with the lazy maximum, below
  // fp16's largest value, and keep 11 bits down to 2^-20 of the row's maximum.
  static constexpr float kLift = 6.f;
  __device__ __forceinline__ static float16_t mma(frag a, frag b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Elem<bf16_t> {
  typedef bf16x8_t frag;
  static constexpr bool kWide = false;
  static constexpr float kLift = 0.f;
  __device__ __forceinline__ static float16_t mma(frag a, frag b, float16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

template <>
struct Elem<float> {
  typedef float8_t frag;
  static constexpr bool kWide = true;
  static constexpr float kLift = 0.f;
  __device__ __forceinline__ static float16_t mma(frag a, frag b, float16_t c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

template <typename T>
using frag_t = typename Elem<T>::frag;

__device__ __forceinline__ float16_t zero16() {
  float16_t z;
#pragma unroll
  for (int r = 0; r < 16; ++r) z[r] = 0.f;
  return z;
}

// Accumulator row of register r in lane half hl (see mfma32 in tj_common.h).
__device__ __forceinline__ constexpr int acc_row(int r, int hl) { return 8 * (r / 4) + 4 * hl + r % 4; }

// Registers 8s .. 8s+7 of an accumulator as the operand fragment that
// contracts its rows 16s .. 16s+15: k-slot (hl, j) stands for accumulator row
// acc_row(8s + j, hl). Rounded to T.
template <typename T>
__device__ __forceinline__ frag_t<T> acc_frag(const float16_t& c, int s) {
  frag_t<T> f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)c[8 * s + j];
  return f;
}

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
template <typename V>
__device__ __forceinline__ V lds_at(uint32_t at) {
  return *(const __attribute__((address_space(3))) V*)(uintptr_t)at;
}

// An LDS tile of rows of W elements without padding. The 16-byte chunk c of a
// row stands at position c ^ swizzle(row), so that what both readers below take
// at a time covers the 64 banks (256 bytes) once: sixteen lanes one chunk of
// sixteen rows, and thirty-two lanes four chunks of four rows.
template <typename T, int W>
struct LdsRows {
  static constexpr int kVec = 16 / (int)sizeof(T);
  static constexpr int kChunks = W / kVec;
  static constexpr int kRowBytes = W * (int)sizeof(T);

  __device__ __forceinline__ static int swizzle(int row) {
    if constexpr (kChunks == 4) return (row >> 2) & 3;
    else if constexpr (kChunks == 8) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return ((row & 3) << 2) | ((row >> 2) & 3);
  }

  // Lane addresses in a tile. A fragment's place is the lane's address with some
  // bits turned (the tile's offset is a multiple of 1024) plus a constant: one
  // register a tile, and one instruction a fragment.
  __device__ __forceinline__ static uint32_t lane_row(int lane) {
    const int row = lane % 32, chunk = (sizeof(T) == 4 ? 2 : 1) * (lane / 32);
    return row * kRowBytes + ((chunk ^ swizzle(row)) << 4);
  }
  __device__ __forceinline__ static uint32_t lane_col(int lane) {
    const int hl = lane / 32;
    if constexpr (sizeof(T) == 4) {
      const int row = 4 * hl, col = lane % 32;
      return row * kRowBytes + (((col / 4) ^ swizzle(row)) << 4) + 4 * (col % 4);
    } else {
      const int row = 4 * hl + (lane & 15) / 4, chunk = (lane & 16) / 8 + (lane & 3) / 2;
      return row * kRowBytes + ((chunk ^ swizzle(row)) << 4) + 8 * (lane & 1);
    }
  }

  // Elements 16 ks + 8 (lane / 32) .. + 7 of row (lane % 32); base: tile +
  // lane_row, offset: rows further on.
  __device__ __forceinline__ static frag_t<T> row_frag(uint32_t base, int ks, int offset) {
    if constexpr (sizeof(T) == 4) {
      const float4_t a = lds_at<float4_t>((base ^ (ks << 6)) + offset);
      const float4_t b = lds_at<float4_t>((base ^ (ks << 6 | 16)) + offset);
      return frag_t<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
      return lds_at<frag_t<T>>((base ^ (ks << 5)) + offset);
    }
  }

  // The fragment that contracts 16 rows in acc_frag's order, for column 32 d +
  // lane % 32; base: tile + lane_col, offset: where the rows start. 16-bit
  // elements come through the transposing LDS read: sixteen lanes name 4 rows x
  // 16 columns, lane j of them gets column j.
  __device__ __forceinline__ static frag_t<T> col_frag(uint32_t base, int d, int offset) {
    if constexpr (sizeof(T) == 4) {
      frag_t<T> f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int row = j / 4 * 8 + j % 4;  // beyond the lane's first
        f[j] = lds_at<float>((base ^ (d << 7) ^ (swizzle(row) << 4)) + offset + row * kRowBytes);
      }
      return f;
    } else {
      typedef short short4_t __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) short4_t lds_short4;
      const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(uintptr_t)((base ^ (d << 6)) + offset));
      const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4*)(uintptr_t)((base ^ (d << 6) ^ (swizzle(8) << 4)) + offset + 8 * kRowBytes));
      return __builtin_bit_cast(frag_t<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// ROWS rows of memory into an LDS tile, by WAVES waves, without registers:
// each instruction brings 64 chunks of 16 bytes to consecutive places, so a
// lane asks for the chunk that belongs at its place. Bounds-checked buffer
// loads: what lies outside the resource, and columns at or past the width, land
// as zeros. The copies are in flight until the wave has waited for them
// (wait_copies) and the workgroup has met.
//
// The copy is an asm statement because the compiler, where it knows of one in
// flight, waits for it before every transposing LDS read, whatever that reads.
// It has no register results, so nothing can be reused too early, and loads the
// compiler does not count only make its own waits stricter (they end in order).
// The wait state between m0's write and its use is in the statement.
constexpr uint32_t kOutside = 0x80000000u;
typedef uint32_t rsrc_t __attribute__((ext_vector_type(4)));

// Raw buffer resource of `bytes` bytes at p (the same in every lane).
__device__ __forceinline__ rsrc_t make_rsrc(const void* p, uint32_t bytes) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  return rsrc_t{(uint32_t)u, (uint32_t)(u >> 32) & 0xffffu, bytes, kDiffBufferFlags};
}

__device__ __forceinline__ void copy_16(rsrc_t r, uint32_t lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(r)
               : "memory", "m0");
}

template <typename T, int W, int ROWS, int WAVES>
struct TileCopy {
  using L = LdsRows<T, W>;
  static constexpr int kRowsPer = 64 / L::kChunks;             // rows of one instruction
  static constexpr int kTotal = ROWS / kRowsPer;               // instructions of the tile
  static constexpr int N = (kTotal + WAVES - 1) / WAVES;       // of one wave
  static_assert(ROWS % kRowsPer == 0 && (kTotal % WAVES == 0 || kTotal < WAVES), "tile rows");

  __device__ __forceinline__ static int row(int wave, int n, int lane) {
    return (wave * N + n) * kRowsPer + lane / L::kChunks;
  }
  // Byte offset of the lane's chunk in its row, outside for columns past `width`.
  __device__ __forceinline__ static uint32_t chunk(int row, int lane, int width) {
    const int c = (lane % L::kChunks) ^ L::swizzle(row);
    return c * L::kVec < width ? (uint32_t)c * 16 : kOutside;
  }
  __device__ __forceinline__ static void issue(rsrc_t r, uint32_t tile, int wave, int n, uint32_t voff) {
    if (kTotal < WAVES && wave >= kTotal) return;
    copy_16(r, tile + (wave * N + n) * 1024, voff);
  }
};

// A tile of consecutive rows (keys), whose lanes' offsets never change: the
// resource moves along.
template <typename T, int W, int ROWS, int WAVES>
struct KeyCopy : TileCopy<T, W, ROWS, WAVES> {
  using C = TileCopy<T, W, ROWS, WAVES>;
  uint32_t voff[C::N];
  __device__ __forceinline__ void init(int64_t row_stride, int width, int wave, int lane) {
#pragma unroll
    for (int n = 0; n < C::N; ++n) {
      const int r = C::row(wave, n, lane);
      const uint32_t c = C::chunk(r, lane, width);
      voff[n] = c == kOutside ? kOutside : (uint32_t)r * (uint32_t)(row_stride * (int64_t)sizeof(T)) + c;
    }
  }
  // Rows 0 .. rows-1 from `p` on to LDS offset `tile`; further rows of the tile read as zeros.
  __device__ __forceinline__ void issue(const T* p, int64_t row_stride, int rows, int width, uint32_t tile, int wave) const {
    const int64_t bytes = rows <= 0 ? 0 : ((int64_t)(min(rows, ROWS) - 1) * row_stride + width) * (int64_t)sizeof(T);
    const rsrc_t r = make_rsrc(p, (uint32_t)bytes);
#pragma unroll
    for (int n = 0; n < C::N; ++n) C::issue(r, tile, wave, n, voff[n]);
  }
};

// 64 single floats the same way: lane l's from byte offset voff to lds + 4 l.
__device__ __forceinline__ void copy_4(rsrc_t r, uint32_t lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds), "v"(voff), "s"(r)
               : "memory", "m0");
}

// N products, the operands of each read from LDS DEPTH products before it. The
// compiler, left to itself, reads right before the use and waits; that is as
// good where other waves fill the gap and the registers are needed (DEPTH 0).
template <int N, int DEPTH, typename Read, typename Use>
__device__ __forceinline__ void read_ahead(Read&& read, Use&& use) {
  decltype(read(0)) f[N];
#pragma unroll
  for (int i = 0; i < DEPTH && i < N; ++i) f[i] = read(i);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (i + DEPTH < N) f[i + DEPTH] = read(i + DEPTH);
    if constexpr (DEPTH > 0) __builtin_amdgcn_sched_barrier(0);
    use(i, f[i]);
    if constexpr (DEPTH > 0) __builtin_amdgcn_sched_barrier(0);
  }
}

// This wave's copies (and loads) and LDS accesses are done.
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// x plus the sum of a fragment's values.
__device__ __forceinline__ float frag_sum(half8_t f, float x) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) x = __builtin_amdgcn_fdot2(half2_t{f[j], f[j + 1]}, half2_t{1, 1}, x, false);
  return x;
}
__device__ __forceinline__ float frag_sum(bf16x8_t f, float x) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 8; j += 2)
    x = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{f[j], f[j + 1]}, bf16x2_t{(__bf16)1.f, (__bf16)1.f}, x, false);
  return x;
}
__device__ __forceinline__ float frag_sum(float8_t f, float x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x += f[j];
  return x;
}

// Eight consecutive elements of a row in memory, zeros at or past `width`.
template <typename T>
__device__ __forceinline__ frag_t<T> load_frag(const T* p, int k, int width) {
  frag_t<T> f;
  if constexpr (sizeof(T) == 4) {
    float4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (p != nullptr && k < width) a = *reinterpret_cast<const float4_t*>(p + k);
    if (p != nullptr && k + 4 < width) b = *reinterpret_cast<const float4_t*>(p + k + 4);
    f = frag_t<T>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)0.f;
    if (p != nullptr && k < width) f = *reinterpret_cast<const frag_t<T>*>(p + k);
  }
  return f;
}

// Four consecutive values, rounded to T.
template <typename T>
__device__ __forceinline__ void store4t(T* p, float a, float b, float c, float d) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4_t*>(p) = float4_t{a, b, c, d};
  } else {
    typedef T t4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<t4*>(p) = t4{(T)a, (T)b, (T)c, (T)d};
  }
}

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

// The parts of few-row sweeps: of at most `per` blocks of 32 keys, in the order of
// the sequences, the same `per` for all of them, so that the waves of a ragged
// batch end together (sixteen sequences of 16384 .. 65536 keys: 254 us, with as
// many parts for each 284). few_slots times `per` cover all blocks for certain,
// and with a part begun by every sequence that is few_slots + B = n_parts of them
// at most; a smaller `per` is taken where its parts, counted, are no more. With
// few_each, that many parts of every sequence, without a look at the others. A
// whole wave calls these.
struct FewParts {
  int b, first;   // sequence, its first part
  int n, keys;    // its parts, and the keys of each
  __device__ __forceinline__ static uint32_t blocks(const DiffArgs& a, int b) {
    return b < a.B ? (uint32_t)(min(a.Sk, max(0, a.len[b])) + 31) / 32 : 0;
  }
  __device__ __forceinline__ static uint32_t wave_sum(uint32_t x) {
#pragma unroll
    for (int s = kWave / 2; s > 0; s >>= 1) x += __shfl_xor(x, s);
    return x;
  }
  __device__ __forceinline__ static uint32_t blocks_per_part(const DiffArgs& a, int lane) {
    if (a.B == 1) return max(1u, (blocks(a, 0) + a.n_parts - 1) / a.n_parts);
    uint32_t sum = 0;
    for (int b = lane; b < a.B; b += kWave) sum += blocks(a, b);
    sum = wave_sum(sum);
    for (uint32_t begun = a.B; begun > 0; begun = begun == (uint32_t)a.B ? begun / 2 : 0) {
      const uint32_t per = max(1u, (sum + a.few_slots + begun - 1) / (a.few_slots + begun));
      uint32_t n = 0;
      for (int b = lane; b < a.B; b += kWave) n += (blocks(a, b) + per - 1) / per;
      if (wave_sum(n) <= (uint32_t)a.n_parts) return per;
    }
    return max(1u, (sum + a.few_slots - 1) / a.few_slots);
  }
  __device__ __forceinline__ void take(const DiffArgs& a, uint32_t per) {
    const uint32_t k = blocks(a, b);
    n = a.few_each != 0 ? min(a.few_each, (int)k) : (int)((k + per - 1) / per);
    keys = n == 0 ? 0 : (int)((k + n - 1) / n) * 32;
  }
  // The sequence that `part` belongs to; false for none.
  __device__ __forceinline__ bool find(const DiffArgs& a, int part, int lane) {
    if (a.few_each != 0) {
      b = part / a.few_each;
      first = b * a.few_each;
      take(a, 1);
      return part - first < n;
    }
    const uint32_t per = blocks_per_part(a, lane);
    if (a.B == 1) {
      b = first = 0;
      take(a, per);
      return part < n;
    }
    uint32_t before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kWave) {
      const uint32_t own = (blocks(a, b0 + lane) + per - 1) / per;
      uint32_t upto = own;
#pragma unroll
      for (int s = 1; s < kWave; s <<= 1) {
        const uint32_t x = __shfl_up(upto, s);
        if (lane >= s) upto += x;
      }
      const uint64_t past = __ballot((uint32_t)part < before + upto);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        b = b0 + at;
        first = (int)(before + __shfl(upto - own, at));
        take(a, per);
        return true;
      }
      before += __shfl(upto, kWave - 1);
    }
    return false;
  }
  // Sequence `seq`'s parts.
  __device__ __forceinline__ void of(const DiffArgs& a, int seq, int lane) {
    if (a.few_each != 0) {
      b = seq;
      first = b * a.few_each;
      return take(a, 1);
    }
    const uint32_t per = blocks_per_part(a, lane);
    uint32_t before = 0;
    for (int x = lane; x < seq; x += kWave) before += (blocks(a, x) + per - 1) / per;
    b = seq;
    first = (int)wave_sum(before);
    take(a, per);
  }
};

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

// The parts (FewParts) for `groups` workgroups of few rows in all, as many as run
// at once: with more, one sequence of 65536 keys takes 49 us instead of 38 (twice
// as many) and sixteen of them 382 instead of 364. At least one more part than
// sequences, for long ones among short; none below 32 keys. Sequences that fill
// the chip by themselves, or too many to look at in every workgroup, get as many
// parts each as they are.
constexpr int kCus = 256, kMostGroups = 8 * kCus;
struct FewPlan {
  int64_t slots, each, total;
};
inline FewPlan few_plan(int64_t B, int64_t Hk, int64_t mtiles, int64_t Sk, int64_t groups) {
  const int64_t tiles = B * Hk * mtiles, blocks = Sk > 0 ? (Sk + 31) / 32 : 1;
  if (B > 2 * kWave || tiles >= groups) {
    int64_t each = groups / tiles;
    if (each < 1) each = 1;
    if (each > blocks) each = blocks;
    return {0, each, B * each};
  }
  int64_t slots = groups / (Hk * mtiles) - B;
  if (slots < B) slots = B;
  if (slots > B * blocks) slots = B * blocks;
  return {slots, 0, slots + B};
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
