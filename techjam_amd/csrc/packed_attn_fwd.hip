// Attention of packed sequences with grouped heads, forward (the mathematics, the
// row numbering and the regions are in grouped_attn.h).
//
// A workgroup = RB waves of NB blocks of 32 rows of one (sequence, key head) times KG
// groups; key tiles of 32 or 64 stream through LDS, dealt to the groups in turn,
// and the groups' sums meet in LDS at the end.
#include "grouped_attn.h"

namespace tj {
namespace {

constexpr int kThreads = 256;

// Four waves: 128 rows where those fill the chip, else 64 with two groups or 32 with four, if two
// tiles for each fit.
template <typename T, int HD, int BLOCKS, int NBT>
struct FwdShape {
  static constexpr int NB = NBT, RB = BLOCKS, KG = 4 / RB, ROWS = 32 * RB * NB;
  static constexpr int BN = KG == 1 && HD * (int)sizeof(T) <= 256 ? 64 : 32;
  using SH = SweepShape<T, HD, BN>;
};
template <typename T, int HD>
constexpr bool groups_fit(int groups) { return groups * SweepShape<T, HD, 32>::W * (int)sizeof(T) <= 1024; }

template <typename T, int HD, int BLOCKS, int NB, bool STATS>
__global__ __launch_bounds__(kThreads, (NB == 1 && HD * (int)sizeof(T) <= 256 ? 2 : 1)) void packed_fwd_kernel(PackedArgs a) {
  using FS = FwdShape<T, HD, BLOCKS, NB>;
  using SH = typename FS::SH;
  using State = SweepState<T, HD, FS::BN, NB, STATS>;
  constexpr int RB = FS::RB, KG = FS::KG, BN = FS::BN, ROWS = FS::ROWS;
  // Two tiles a group; afterwards the groups' results.
  constexpr int kSums = KG > 1 ? 16 * State::kGive * NB * RB * (KG / 2) : 0;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[KG * 2 * SH::kBytes > kSums ? KG * 2 * SH::kBytes : kSums];
  __shared__ float ml[KG > 1 ? KG / 2 * RB * NB * State::kMl * kWave : 1];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int kg = w / RB, rb = w % RB;
  // Consecutive ids run on the XCDs in turn, so the key head varies fastest: the tiles that share
  // K and V also share an XCD's L2.
  const int hk = blockIdx.x % a.Hk;
  Region g;
  if (!g.take(a, blockIdx.x / a.Hk, a.G, ROWS, false, lane)) return;
  const int L = g.len, R = g.rows * a.G, r0 = g.tile * ROWS, rw0 = r0 + 32 * NB * rb;
  // Keys needed by rows row .. last (clipped to the region's).
  auto span = [&](int row, int last) {
    return row >= R || row / a.G >= L ? 0 : (a.causal ? min(L, min(last, R - 1) / a.G + 1) : L);
  };
  const int kv_end = span(r0, r0 + ROWS - 1), own_end = span(rw0, rw0 + 32 * NB - 1);
  const uint32_t tiles = lds_offset(smem) + kg * 2 * SH::kBytes;
  SweepTiles<T, SH, RB> keys;
  keys.init(reinterpret_cast<const T*>(a.k) + a.vk.row(g.start, hk), reinterpret_cast<const T*>(a.v) + a.vv.row(g.start, hk),
            a.vk.st, a.vv.st, a.D, a.Dv, rb, lane);
  int kv0 = BN * kg;
  if (kv0 < kv_end) keys.issue(kv0, L, tiles, rb);
  State st;
  st.init(a.scale, lane);
  SweepRow row[NB];
  int free[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int first = rw0 + 32 * n, r = first + lane % 32;
    row[n] = SweepRow{r, r / a.G, r % a.G, 0, r < R && r / a.G < L};
    row[n].limit = a.causal ? row[n].i : L - 1;
    free[n] = a.causal ? first / a.G : L - 1;
    st.load_q(n, row[n].live ? reinterpret_cast<const T*>(a.q) + a.vq.row(g.start + row[n].i, hk * a.G + row[n].g) : nullptr,
              a.scale, a.D, lane);
  }
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
        st.step(tiles + cur * SH::kBytes, kb, [&](int n, float16_t& s) {
          if (at + 31 <= free[n]) return;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (at + acc_row(r, lane / 32) > row[n].limit) s[r] = -__builtin_inff();
        });
    }
  }
  // The groups' states, the upper half's joined to the lower half's.
#pragma unroll
  for (int half = KG / 2; half > 0; half /= 2) {
    float4_t* x = reinterpret_cast<float4_t*>(smem);
    const int at = (kg % half) * RB + rb;
    __syncthreads();
    if (kg >= half && kg < 2 * half) st.give(x + at * NB * State::kGive, ml + at * NB * State::kMl * kWave, lane);
    __syncthreads();
    if (kg < half) st.take(x + at * NB * State::kGive, ml + at * NB * State::kMl * kWave, lane);
  }
  if (kg != 0) return;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float inv = 1.f / pair_sum(st.l[n]);
    const float exact = STATS ? pair_sum(st.e[STATS ? n : 0]) : 0.f;
    if (row[n].r >= R) continue;
    const int64_t token = g.start + row[n].i;
    const int head = hk * a.G + row[n].g;
    if (STATS && row[n].live && lane < 32) a.lse[token * a.H + head] = st.m[n] - Elem<T>::kLift + log2f(exact);
    T* op = reinterpret_cast<T*>(a.o) + a.vo.row(token, head);
    T* rp = reinterpret_cast<T*>(a.rest) + a.vo.row(token, head);
    st.columns(n, a.Dv, lane, [&](int col, float4_t y) {
      if (!row[n].live) y = float4_t{0.f, 0.f, 0.f, 0.f};
      else y *= inv;
      store4t<T>(op + col, y[0], y[1], y[2], y[3]);
      if constexpr (STATS && sizeof(T) == 2)
        store4t<T>(rp + col, y[0] - (float)(T)y[0], y[1] - (float)(T)y[1], y[2] - (float)(T)y[2], y[3] - (float)(T)y[3]);
    });
  }
}

template <typename T, int HD, int BLOCKS, int NB>
int launch(PackedArgs a, hipStream_t stream) {
  constexpr int ROWS = FwdShape<T, HD, BLOCKS, NB>::ROWS;
  const int64_t slots = region_slots(a.T, a.N, a.G, ROWS);
  a.n_slots = (int)slots;
  const dim3 grid(uint32_t(slots * a.Hk));
  if (a.lse != nullptr) hipLaunchKernelGGL((packed_fwd_kernel<T, HD, BLOCKS, NB, true>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((packed_fwd_kernel<T, HD, BLOCKS, NB, false>), grid, dim3(kThreads), 0, stream, a);
  return tjh::launch_status();
}

}  // namespace

int packed_fwd(const PackedArgs& a, int dtype, hipStream_t stream) {
  return grouped_dispatch(a.D, a.Dv, dtype, [&](auto t, auto hd) {
    using T = decltype(t);
    constexpr int HD = decltype(hd)::value;
    const int64_t rows = (int64_t)a.T * a.G;  // of one key head
    if constexpr (groups_fit<T, HD>(4))
      if ((rows + 63) / 64 * a.Hk <= kCus / 2) return launch<T, HD, 1, 1>(a, stream);
    if constexpr (groups_fit<T, HD>(2))
      if ((rows + 127) / 128 * a.Hk <= kCus) return launch<T, HD, 2, 1>(a, stream);
    return launch<T, HD, 4, 1>(a, stream);
  });
}

}  // namespace tj
