// Attention of drafted tokens against a cache, with grouped heads (the mathematics
// and the row numbering are in grouped_attn.h). The Sq drafted tokens of a sequence
// stand in its cache behind what it has settled, at positions len - Sq on; token t sees
// all settled keys, and of the drafted ones its own and those on its line of parents.
//
// A workgroup = RB waves of 32 rows of one (sequence, key head) times KG groups over one
// part of the keys, so that up to 256 rows read a key from memory once; the tiles are dealt to the
// groups, whose sums meet in LDS at the end. Parts are joined by tree_join_kernel.
//
// Medians of a hundred calls after two hundred others. Bound by the cache's bytes: 8 sequences of 22528 to 65536 keys, 16
// drafts, 16 heads on 4, 128 dims, bf16: 132 us + 6 of joining, 5.5 TB/s (a copy of 1 GiB: 5.1); 64 sequences of 1072 to 4096
// keys, one token, 64 dims, fp16: 31 us + 4, 5.5 TB/s. 256 rows a key head (64 drafts, 16 sequences of up to 8192 keys) take
// 58 us, 3.2 TB/s: every part leaves 128 KB of sums, 34 MB in all, written in 7 us and joined in 9.
#include "grouped_attn.h"

namespace tj {
namespace {

constexpr int kJoinThreads = 256;

// The drafted tokens that each one sees, a bit each: the line of parents is followed in
// steps of twice the length, token t in lane t, six times for up to 64 of them. A token
// is not there when its parent does not stand before it, when its position is negative,
// or when something on its line is not there.
struct Lineage {
  uint64_t seen;
  bool gone;
  __device__ __forceinline__ Lineage(const TreeArgs& a, int b, int ctx, int lane) {
    const int p = lane < a.Sq ? a.parents[(int64_t)b * a.Sq + lane] : lane;
    gone = p < -1 || p >= lane || ctx + lane < 0;
    seen = uint64_t(1) << lane;
    int up = gone ? -1 : p;
#pragma unroll
    for (int s = 0; s < 6; ++s) {
      const int from = max(up, 0);
      const uint32_t lo = __shfl((uint32_t)seen, from), hi = __shfl((uint32_t)(seen >> 32), from);
      const int next = __shfl(up, from), lost = __shfl((int)gone, from);
      if (up >= 0) {
        seen |= (uint64_t)hi << 32 | lo;
        gone |= lost != 0;
        up = next;
      }
    }
  }
};

// Four waves of key groups for up to 64 rows, so that four parts meet in LDS rather than in memory; eight
// waves in all at the most, and two tiles a group in at most 128 KB.
template <typename T, int HD, int BLOCKS>
struct TreeShape {
  static constexpr int RB = BLOCKS, ROWS = 32 * RB, BN = RB == 8 ? 64 : 32;
  using SH = SweepShape<T, HD, BN>;
  static constexpr int kFit = 128 * 1024 / (2 * SH::kBytes), kMost = RB <= 2 ? 4 : 8 / RB, KG = kFit < kMost ? kFit : kMost;
  static constexpr int WAVES = RB * KG, THREADS = kWave * WAVES;
  using Wave = WaveRows<T, HD>;
  // Two tiles a group, afterwards the groups' results.
  static constexpr int kTiles = KG * 2 * SH::kBytes, kSums = KG > 1 ? 16 * SH::DB * 4 * kWave * RB * (KG / 2) : 0;
  static constexpr int kBytes = kTiles > kSums ? kTiles : kSums;
  // q comes through the second tile while the first keys are on their way, or before them where it needs both.
  static constexpr bool kBefore = RB * Wave::kBytes > SH::kBytes;
  static_assert(RB * Wave::kBytes <= 2 * SH::kBytes, "room for q");
  // Waves of a SIMD by the registers, and workgroups that a CU holds.
  static constexpr int kWaves = HD == 32 ? 3 : (sizeof(T) == 2 || HD == 64 || WAVES > 4 ? 2 : 1);
  static constexpr int kByLds = 160 * 1024 / kBytes, kByRegs = kWaves * 4 / WAVES;
  static constexpr int kPerCu = kByLds < kByRegs ? kByLds : kByRegs;
  static_assert(kPerCu >= 1, "a workgroup fits a CU");
};

template <typename T, int HD, int BLOCKS>
__global__ __launch_bounds__((TreeShape<T, HD, BLOCKS>::THREADS), (TreeShape<T, HD, BLOCKS>::kWaves)) void tree_kernel(TreeArgs a) {
  using TS = TreeShape<T, HD, BLOCKS>;
  using SH = typename TS::SH;
  using State = SweepState<T, HD, TS::BN, false>;
  constexpr int RB = TS::RB, KG = TS::KG, BN = TS::BN;
  using Wave = typename TS::Wave;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[TS::kBytes];
  __shared__ float ml[KG > 1 ? KG / 2 * RB * State::kMl * kWave : 1];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int kg = w / RB, rb = w % RB;
  const int mt = blockIdx.x % a.n_mtiles, hk = blockIdx.x / a.n_mtiles % a.Hk, part = blockIdx.x / a.n_mtiles / a.Hk;
  const bool whole = a.part_o == nullptr;
  FewParts f;
  if (whole) f.b = part;
  else if (!f.find(a, part, lane)) return;
  const int b = __builtin_amdgcn_readfirstlane(f.b);
  // For the join, which need not count parts again.
  if (!whole && part == f.first && hk == 0 && mt == 0 && tid == 0) {
    a.plan[2 * b] = f.first;
    a.plan[2 * b + 1] = f.keys;
  }
  const int L = __builtin_amdgcn_readfirstlane(min(a.Sk, max(0, a.len[b]))), ctx = L - a.Sq;
  const int row0 = mt * TS::ROWS, rw0 = row0 + 32 * rb;
  // Keys that rows row .. last (clipped to R) need.
  auto span = [&](int row, int last) { return row >= a.R ? 0 : max(0, ctx + min(last, a.R - 1) / a.by_group + 1); };
  const int n_keys = whole ? L : __builtin_amdgcn_readfirstlane(f.keys);
  const int kv_begin = whole ? 0 : __builtin_amdgcn_readfirstlane((part - f.first) * f.keys);
  const int kv_end = min(span(row0, row0 + TS::ROWS - 1), kv_begin + n_keys), own_end = min(kv_end, span(rw0, rw0 + 31));
  if (kv_begin >= kv_end && !whole) return;  // not read either
  const uint32_t tiles = lds_offset(smem) + kg * 2 * SH::kBytes;
  SweepTiles<T, SH, RB> keys;
  keys.init(reinterpret_cast<const T*>(a.k) + a.vk.row(b, hk, 0), reinterpret_cast<const T*>(a.v) + a.vv.row(b, hk, 0),
            a.vk.ss, a.vv.ss, a.D, a.Dv, rb, lane);
  int kv0 = kv_begin + BN * kg;
  if (!TS::kBefore && kv0 < kv_end) keys.issue(kv0, L, tiles, rb);
  const int r = rw0 + lane % 32;
  SweepRow row{r / a.by_group, r % a.by_group, 0, false};
  row.limit = ctx + row.i;
  row.live = r < a.R && row.limit >= 0;
  uint64_t seen = 0, gone = 0;
  if (a.parents != nullptr) {
    const Lineage line(a, b, ctx, lane);
    const int t = min(row.i, kWave - 1);
    seen = (uint64_t)__shfl((uint32_t)(line.seen >> 32), t) << 32 | (uint64_t)__shfl((uint32_t)line.seen, t);
    gone = __ballot(line.gone && lane < a.Sq);
    row.live = row.live && !(gone >> t & 1);
  }
  State st;
  const typename Wave::Places places(rw0, a.by_group, lane);
  const int token0 = rw0 / a.by_group;
  {
    typename Wave::vec_t x[Wave::N];
    Wave::read(x, reinterpret_cast<const T*>(a.q) + a.vq.row(b, hk * a.G, token0), a.vq.ss, a.vq.sh, a.D, places, a.R, lane);
    Wave::turn(x, tiles + (TS::kBefore ? 0 : SH::kBytes) + rb * Wave::kBytes, lane, st.q);
  }
  if constexpr (TS::kBefore) {
    __syncthreads();
    if (kv0 < kv_end) keys.issue(kv0, L, tiles, rb);
  }
  st.init(a.scale, lane);
  // The workgroup goes round together, the last round maybe without a tile for every group.
  for (int first = kv_begin, cur = 0; first < kv_end; first += KG * BN, kv0 += KG * BN, cur ^= 1) {
    // The tile is there, and the group's other one has been read by its waves. (A group of one wave has waited for
    // itself.)
    wait_copies();
    if constexpr (RB > 1) lds_barrier();
    if (kv0 + KG * BN < kv_end) keys.issue(kv0 + KG * BN, L, tiles + (cur ^ 1) * SH::kBytes, rb);
    const uint32_t tile = tiles + cur * SH::kBytes;
    if (gone != 0 && first + KG * BN > ctx) {
      // What is not there may hold anything: its values are cleared, as 0 times NaN would spoil the others.
      constexpr int kChunks = SH::Rows::kChunks;
      for (int c = rb * kWave + lane; c < BN * kChunks; c += RB * kWave) {
        const int t = kv0 + c / kChunks - ctx;
        if (t >= 0 && t < kWave && (gone >> t & 1))
          *(__attribute__((address_space(3))) float4_t*)(uintptr_t)(tile + SH::kTensor + c * 16) = float4_t{0.f, 0.f, 0.f, 0.f};
      }
      wait_lds();
      if constexpr (RB > 1) lds_barrier();
    }
#pragma unroll
    for (int kb = 0; kb < BN / 32; ++kb) {
      const int at = kv0 + 32 * kb;
      if (at >= own_end) continue;
      st.step(tile, kb, [&](float16_t& s) {
        const int hl = lane / 32;
        if (at + 32 <= ctx) return;
        if (a.parents == nullptr) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (at + acc_row(e, hl) > row.limit) s[e] = -__builtin_inff();
          return;
        }
        // The 32 keys that the row sees: settled ones, then its line.
        const int t = at - ctx;  // drafted token of the first key
        uint32_t word = t >= kWave ? 0 : (t >= 0 ? (uint32_t)(seen >> t) : (uint32_t)(seen << -t) | ((1u << -t) - 1));
        word >>= 4 * hl;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(word >> acc_row(e, 0) & 1)) s[e] = -__builtin_inff();
      });
    }
  }
  // The groups' states, the upper half's joined to the lower half's.
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    float4_t* x = reinterpret_cast<float4_t*>(smem) + ((kg % half) * RB + rb) * State::kGive;
    float* y = ml + ((kg % half) * RB + rb) * State::kMl * kWave;
    __syncthreads();
    if (kg >= half && kg < 2 * half) st.give(x, y, lane);
    __syncthreads();
    if (kg < half) st.take(x, y, lane);
  }
  __syncthreads();  // the tiles, in whose place the rows are turned, have been read
  const float sum = pair_sum(st.l);
  if (kg != 0) return;
  if (whole) {
    const float inv = 1.f / sum;
    Wave::write(reinterpret_cast<T*>(a.o) + a.vo.row(b, hk * a.G, token0), a.vo.ss, a.vo.sh, a.Dv, places, a.R,
                lds_offset(smem) + rb * Wave::kBytes, lane,
                [&](int d, int c) { return row.live ? st.four(d, c) * inv : float4_t{0.f, 0.f, 0.f, 0.f}; });
    return;
  }
  if (r >= a.R) return;
  const int64_t at = ((int64_t)part * a.Hk + hk) * a.R + r;
  if (lane < 32) *reinterpret_cast<float4_t*>(a.part_ml + at * 4) = float4_t{st.m, sum, row.live ? 1.f : 0.f, 0.f};
  if (!row.live) return;
#pragma unroll
  for (int d = 0; d < SH::DB; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int col = 32 * d + 8 * c + 4 * (lane / 32);
      if (col < a.Dv) *reinterpret_cast<float4_t*>(a.part_o + at * a.Dv + col) = st.four(d, c);
    }
}

// Joins the parts: O = sum_p 2^(max_p - M) o_p / sum_p 2^(max_p - M) sum_p. `lanes` threads take a row's
// chunks of 4 columns, `sets` of them every so many-th part, the workgroup's 256 threads as many rows as
// that leaves. A row's parts are those up to its last key.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void tree_join_kernel(TreeArgs a, int lanes, int sets) {
  __shared__ float4_t part[kJoinThreads];
  __shared__ float top[kJoinThreads], total[kJoinThreads];
  const int tid = threadIdx.x, per_row = lanes * sets, rows = kJoinThreads / per_row;
  const int chunk = tid % lanes, set = tid / lanes % sets;
  const int tiles = (a.R + rows - 1) / rows;  // of one (sequence, key head)
  const int bh = blockIdx.x / tiles, b = bh / a.Hk, hk = bh % a.Hk;
  const int r = blockIdx.x % tiles * rows + tid / per_row, i = r / a.by_group;
  const int L = min(a.Sk, max(0, a.len[b])), limit = L - a.Sq + i;
  int np = 0;
  int64_t at = 0;  // the row's number in its first part
  if (r < a.R && limit >= 0) {
    np = limit / a.plan[2 * b + 1] + 1;
    at = ((int64_t)a.plan[2 * b] * a.Hk + hk) * a.R + r;
  }
  const int64_t step = (int64_t)a.Hk * a.R;
  const bool on = chunk * 4 < a.Dv;
  float m = -__builtin_inff(), l = 0.f, live = 0.f;
  float4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = set; p < np; p += sets) {
    const float4_t x = *reinterpret_cast<const float4_t*>(a.part_ml + (at + p * step) * 4);
    const float4_t o = *reinterpret_cast<const float4_t*>(a.part_o + (at + p * step) * a.Dv + (on ? chunk : 0) * 4);
    live = x[2];
    const float to = fmaxf(m, x[0]);
    // An unset maximum (-inf) goes with sums that are zero, or NaN and kept.
    const float w0 = m == -__builtin_inff() ? 1.f : fast_exp2(m - to), w1 = x[0] == -__builtin_inff() ? 1.f : fast_exp2(x[0] - to);
    m = to;
    l = fmaf(l, w0, x[1] * w1);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaf(y[j], w0, o[j] * w1);
  }
  part[tid] = y;
  top[tid] = m;
  total[tid] = l;
  __syncthreads();
  if (set != 0 || r >= a.R || !on) return;
  float most = m;
  for (int s = 1; s < sets; ++s) most = fmaxf(most, top[tid + s * lanes]);
  const float w0 = m == -__builtin_inff() ? 1.f : fast_exp2(m - most);
  l *= w0;
  y *= w0;
  for (int s = 1; s < sets; ++s) {
    const float x = top[tid + s * lanes], w = x == -__builtin_inff() ? 1.f : fast_exp2(x - most);
    const float4_t o = part[tid + s * lanes];
    l = fmaf(total[tid + s * lanes], w, l);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaf(o[j], w, y[j]);
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = live != 0.f ? y[j] * inv : 0.f;
  store4t<T>(reinterpret_cast<T*>(a.o) + a.vo.row(b, hk * a.G + r % a.by_group, i) + chunk * 4, y[0], y[1], y[2], y[3]);
}

template <typename T>
int launch_join(const TreeArgs& a, hipStream_t stream) {
  int lanes = 1, sets = 1;
  while (lanes * 4 < a.Dv) lanes *= 2;
  // As many sets as leave each a part or two, but not more threads than run at once (16384 rows of five parts:
  // 12.2 us with two sets, 8.6 with one; 2048 rows of 40 parts: 6.0 with eight, 6.9 with half as many rows a workgroup).
  const int parts = a.few_each != 0 ? a.few_each : (a.n_parts + a.B - 1) / a.B;
  const int64_t threads = (int64_t)a.B * a.Hk * a.R * lanes;
  while (2 * sets < parts && lanes * sets < kJoinThreads && threads * sets < (1 << 19)) sets *= 2;
  const int rows = kJoinThreads / (lanes * sets), tiles = (a.R + rows - 1) / rows;
  hipLaunchKernelGGL((tree_join_kernel<T>), dim3(uint32_t((int64_t)a.B * a.Hk * tiles)), dim3(kJoinThreads), 0, stream, a, lanes, sets);
  return tjh::launch_status();
}

template <typename T, int HD, int BLOCKS>
int launch(const TreeArgs& a, hipStream_t stream) {
  using TS = TreeShape<T, HD, BLOCKS>;
  const int64_t parts = a.part_o == nullptr ? a.B : a.n_parts;
  hipLaunchKernelGGL((tree_kernel<T, HD, BLOCKS>), dim3(uint32_t(parts * a.Hk * a.n_mtiles)), dim3(TS::THREADS), 0, stream, a);
  const int rc = tjh::launch_status();
  return rc != TJ_OK || a.part_o == nullptr ? rc : launch_join<T>(a, stream);
}

// f(integral_constant<int, blocks of 32 rows a workgroup>); eight blocks of fp32 rows spill.
template <typename T, typename F>
auto by_blocks(int R, F&& f) {
  if (R <= 32) return f(std::integral_constant<int, 1>{});
  if (R <= 64) return f(std::integral_constant<int, 2>{});
  if constexpr (sizeof(T) == 2)
    if (R > 128) return f(std::integral_constant<int, 8>{});
  return f(std::integral_constant<int, 4>{});
}

}  // namespace

TreePlan tree_plan(const TreeArgs& a, int dtype) {
  TreePlan p{};
  grouped_dispatch(a.D, a.Dv, dtype, [&](auto t, auto hd) {
    by_blocks<decltype(t)>(a.R, [&](auto blocks) {
      using TS = TreeShape<decltype(t), decltype(hd)::value, decltype(blocks)::value>;
      p.blocks = TS::RB;
      // Short caches are swept whole, in eight rounds at the most: one launch, 10.4 us, instead of 6.7 + 4.9 and the gap
      // between (one sequence of 1024 keys, 8 heads, 64 dims).
      if (a.Sk <= 8 * TS::KG * TS::BN) p.parts = FewPlan{0, 1, a.B};
      else p.parts = few_plan(a.B, a.Hk, (a.R + TS::ROWS - 1) / TS::ROWS, a.Sk, kCus * TS::kPerCu);
      return 0;
    });
    return 0;
  });
  return p;
}

int tree_fwd(const TreeArgs& args, const TreePlan& p, int dtype, hipStream_t stream) {
  TreeArgs a = args;
  a.n_mtiles = (a.R + 32 * p.blocks - 1) / (32 * p.blocks);
  a.few_slots = (int)p.parts.slots;
  a.few_each = (int)p.parts.each;
  a.n_parts = (int)p.parts.total;
  return grouped_dispatch(a.D, a.Dv, dtype, [&](auto t, auto hd) {
    return by_blocks<decltype(t)>(a.R, [&](auto blocks) {
      return launch<decltype(t), decltype(hd)::value, decltype(blocks)::value>(a, stream);
    });
  });
}

}  // namespace tj
