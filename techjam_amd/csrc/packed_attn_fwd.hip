// Attention of packed sequences with grouped heads, forward (the mathematics, the
// row numbering and the regions are in grouped_attn.h).
//
// A workgroup = RB waves of 32 rows of one (sequence, key head) times KG
// groups; key tiles of 32 or 64 stream through LDS, dealt to the groups in turn,
// and the groups' sums meet in LDS at the end.
//
// Medians of a hundred calls after two hundred others. Long sequences are bound by power: 32768 tokens, 8 heads on 2,
// 128 dims, bf16, causal take 2032 us (1906 on another card), 1082 TFLOP/s of 2D + 2Dv operations a pair (a large
// library product of that type 1218), the matrix unit 59 % and the vector unit 52 % busy at a clock of 1.72 of 2.4 GHz.
// Short ones are bound by what stands before and after their few key tiles: 96 sequences of about 340
// tokens, 16 heads on 4, 64 dims take 86 us, of which looking for the tile, q, and the results
// take 47 without any keys (235 MB, 5 TB/s), the vector unit 61 % busy. A batch of 24 prompts of up to
// 2935 tokens, 16384 in all, 16 heads on 2, 128 dims: 115 us. It is balanced (dealt to the 512 places of two workgroups
// a CU, the 2068 tiles end after 47 rounds of 64 keys where the mean is 46), so a pair of rounds takes 2.4 us of a CU whose
// matrix units need 0.9: with two waves a SIMD a wave's scores, exponentials and values follow each other.
#include "grouped_attn.h"

namespace tj {
namespace {

constexpr int kThreads = 256;

// Four waves: 128 rows where those fill the chip (two workgroups a CU past 64 dims, by the LDS, else
// four), else 64 with two groups or 32 with four, if two tiles for each fit. us with 128 / 64 rows: 512 tiles of 128 rows, 64
// dims 24 / 19, 4260 tiles 92 / 121; 423 tiles of 96 dims 24 / 28, 2068 of 128 dims 120 / 163. Long causal sequences want them
// up to twice as far, as tiles that all run at once end when the longest does: 512 tiles of 128 dims of 16384 tokens
// 463 / 356, of 4096 112 / 97, but of 1024 37 / 40 and of 256 20 / 27; 768 of 64 dims of 16384 316 / 288.
template <typename T, int HD, int BLOCKS>
struct FwdShape {
  static constexpr int RB = BLOCKS, KG = 4 / RB, ROWS = 32 * RB;
  static constexpr int BN = KG == 1 && HD * (int)sizeof(T) <= 256 ? 64 : 32;
  using SH = SweepShape<T, HD, BN>;
  using State = SweepState<T, HD, BN, true>;
  using Wave = WaveRows<T, HD>;
  // Two tiles a group, afterwards the groups' results.
  static constexpr int kTiles = KG * 2 * SH::kBytes, kSums = KG > 1 ? 16 * State::kGive * RB * (KG / 2) : 0;
  static constexpr int kBytes = kTiles > kSums ? kTiles : kSums;
  // q comes through the second tile while the first keys are on their way, or before them where it needs both.
  static constexpr bool kBefore = RB * Wave::kBytes > SH::kBytes;
  static_assert(RB * Wave::kBytes <= 2 * SH::kBytes, "room for q");
};
template <typename T, int HD>
constexpr bool groups_fit(int groups) { return groups * SweepShape<T, HD, 32>::W * (int)sizeof(T) <= 1024; }

template <typename T, int HD, int BLOCKS, bool STATS>
__global__ __launch_bounds__(kThreads, (HD * (int)sizeof(T) <= 256 ? 2 : 1)) void packed_fwd_kernel(PackedArgs a) {
  using FS = FwdShape<T, HD, BLOCKS>;
  using SH = typename FS::SH;
  using Wave = typename FS::Wave;
  using State = SweepState<T, HD, FS::BN, STATS>;
  constexpr int RB = FS::RB, KG = FS::KG, BN = FS::BN, ROWS = FS::ROWS;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[FS::kBytes];
  __shared__ float ml[KG > 1 ? KG / 2 * RB * State::kMl * kWave : 1];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int kg = w / RB, rb = w % RB;
  // Consecutive ids run on the XCDs in turn, so the key head varies fastest: the tiles that share
  // K and V also share an XCD's L2.
  const int hk = blockIdx.x % a.Hk;
  __shared__ int told[6];
  Region g;
  if (!g.take(a, blockIdx.x / a.Hk, a.G, ROWS, false, tid, told)) return;
  const int L = g.len, R = g.rows * a.G, r0 = g.tile * ROWS, rw0 = r0 + 32 * rb;
  // Keys needed by rows row .. last (clipped to the region's).
  auto span = [&](int row, int last) {
    return row >= R || row / a.by_group >= L ? 0 : (a.causal ? min(L, min(last, R - 1) / a.by_group + 1) : L);
  };
  const int kv_end = span(r0, r0 + ROWS - 1), own_end = span(rw0, rw0 + 31);
  const uint32_t tiles = lds_offset(smem) + kg * 2 * SH::kBytes;
  SweepTiles<T, SH, RB> keys;
  keys.init(reinterpret_cast<const T*>(a.k) + a.vk.row(g.start, hk), reinterpret_cast<const T*>(a.v) + a.vv.row(g.start, hk),
            a.vk.st, a.vv.st, a.D, a.Dv, rb, lane);
  int kv0 = BN * kg;
  if (!FS::kBefore && kv0 < kv_end) keys.issue(kv0, L, tiles, rb);
  const typename Wave::Places places(rw0, a.by_group, lane);
  const int64_t token0 = g.start + rw0 / a.by_group;
  State st;
  {
    typename Wave::vec_t x[Wave::N];
    Wave::read(x, reinterpret_cast<const T*>(a.q) + a.vq.row(token0, hk * a.G), a.vq.st, a.vq.sh, a.D, places, L * a.G, lane);
    Wave::turn(x, tiles + (FS::kBefore ? 0 : SH::kBytes) + rb * Wave::kBytes, lane, st.q);
  }
  if constexpr (FS::kBefore) {
    __syncthreads();
    if (kv0 < kv_end) keys.issue(kv0, L, tiles, rb);
  }
  st.init(a.scale, lane);
  const int r = rw0 + lane % 32;
  SweepRow row{r / a.by_group, r % a.by_group, 0, r < R && r / a.by_group < L};
  row.limit = a.causal ? row.i : L - 1;
  const int free = a.causal ? rw0 / a.by_group : L - 1;  // the last key that all of the wave's rows see
  // The workgroup goes round together, the last round maybe without a tile for every group.
  for (int first = 0, cur = 0; first < kv_end; first += KG * BN, kv0 += KG * BN, cur ^= 1) {
    // The tile is there, and the group's other one has been read by its waves.
    wait_copies();
    lds_barrier();
    if (kv0 + KG * BN < kv_end) keys.issue(kv0 + KG * BN, L, tiles + (cur ^ 1) * SH::kBytes, rb);
#pragma unroll
    for (int kb = 0; kb < BN / 32; ++kb) {
      const int at = kv0 + 32 * kb;
      if (at < own_end)
        st.step(tiles + cur * SH::kBytes, kb, [&](float16_t& s) {
          if (at + 31 <= free) return;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (at + acc_row(r, lane / 32) > row.limit) s[r] = -__builtin_inff();
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
  if (kg != 0) return;
  const float inv = 1.f / pair_sum(st.l);
  if constexpr (STATS) {
    const float exact = pair_sum(st.e);
    if (row.live && lane < 32) a.lse[(int64_t)(g.start + row.i) * a.H + hk * a.G + row.g] = st.m - Elem<T>::kLift + log2f(exact);
  }
  const uint32_t turn = lds_offset(smem) + rb * Wave::kBytes;
  auto value = [&](int d, int c) { return row.live ? st.four(d, c) * inv : float4_t{0.f, 0.f, 0.f, 0.f}; };
  const int64_t at = a.vo.row(token0, hk * a.G);
  Wave::write(reinterpret_cast<T*>(a.o) + at, a.vo.st, a.vo.sh, a.Dv, places, R, turn, lane, value);
  if constexpr (STATS && sizeof(T) == 2) {
    wait_lds();
    Wave::write(reinterpret_cast<T*>(a.rest) + at, a.vo.st, a.vo.sh, a.Dv, places, R, turn, lane, [&](int d, int c) {
      float4_t y = value(d, c);
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = (y[j] - (float)(T)y[j]) * kRestLift<T>;
      return y;
    });
  }
}

template <typename T, int HD, int BLOCKS>
int launch(PackedArgs a, hipStream_t stream) {
  constexpr int ROWS = FwdShape<T, HD, BLOCKS>::ROWS;
  const int64_t slots = region_slots(a.T, a.N, a.G, ROWS);
  a.n_slots = (int)slots;
  const dim3 grid(uint32_t(slots * a.Hk));
  if (a.lse != nullptr) hipLaunchKernelGGL((packed_fwd_kernel<T, HD, BLOCKS, true>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((packed_fwd_kernel<T, HD, BLOCKS, false>), grid, dim3(kThreads), 0, stream, a);
  return tjh::launch_status();
}

}  // namespace

int packed_fwd(const PackedArgs& a, int dtype, hipStream_t stream) {
  return grouped_dispatch(a.D, a.Dv, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    const int64_t rows = (int64_t)a.T * a.G;  // of one key head
    if constexpr (groups_fit<T, HD>(4))
      if ((rows + 63) / 64 * a.Hk <= kCus / 2) return launch<T, HD, 1>(a, stream);
    if constexpr (groups_fit<T, HD>(2))
      if ((rows + 127) / 128 * a.Hk <= (HD <= 64 ? 2 : 1) * (long_triangles(a) ? 2 : 1) * kCus) return launch<T, HD, 2>(a, stream);
    return launch<T, HD, 4>(a, stream);
  });
}

}  // namespace tj
