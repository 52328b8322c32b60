// Differential attention: the C ABI entry points, their argument checks and
// the choice between one sweep over the keys and parts of it. The kernels are in
// diff_attn_fwd.hip, diff_attn_bwd_kv.hip and diff_attn_bwd_q.hip.
#include "diff_attn.h"

namespace tj {

int diff_delta(const DiffArgs& a, int dtype, hipStream_t stream);

namespace {

int elem_bytes(int dtype) { return dtype == TJ_F32 ? 4 : (dtype == TJ_F16 || dtype == TJ_BF16 ? 2 : 0); }

// How a forward call runs: 32-row waves on their own (few rows) or workgroups of
// 64 or 128 rows; n_parts as in DiffArgs, the most a few-row kernel asks for.
struct DiffPlan {
  bool few;
  int64_t n_parts;
};

// Rows of one key head up to which every wave works by itself, so that the parts of the
// keys follow the batch's lengths. us by waves / by workgroups, 16 sequences against caches
// of 65536, 4 key heads, d64 bf16: lengths spread over a factor of four, 4 rows 249 / 270, 32
// rows 265 / 286, 64 rows 455 / 320; one long sequence among short ones 40 / 153, 45 / 156,
// 70 / 216. Past 64 rows the waves read the keys too often: spread to 16384, 80 rows 188 / 140,
// 256 rows 520 / 300. (Even lengths alone would have the border lower: 64 sequences of 2048
// and fewer, 8 key heads, 16 rows 104 / 71.)
constexpr int64_t kFewRows = 64;

// More rows than few: parts of at least kPartKeys keys where workgroups of 64 rows
// leave half of the CUs idle, as many as fill them (twice where two fit a CU). They cost
// the join of every row, so only from kPartsFrom keys on. Forward, us with parts / without:
// b1 h2 s4096 d64 bf16 57 / 81, h1 s8192 79 / 153, h4 s2048 49 / 47, fp32 142 / 225; 512 new
// rows a key head against 4096 keys 32 / 82; with 256 workgroups already, h8 s2048 75 / 48.
constexpr int64_t kPartsFrom = 2048;
DiffPlan plan(int64_t B, int64_t Hk, int64_t R, int64_t Sk, int64_t Dv, bool cached) {
  if (cached && R <= kFewRows) return {true, few_plan(B, Hk, (R + 31) / 32, Sk, kMostGroups).total};
  const int64_t tiles = B * Hk * ((R + 63) / 64);
  if (tiles > kCus / 2 || Sk < kPartsFrom) return {false, 1};
  const int64_t fill = Dv > 128 ? kCus : 2 * kCus, want = (fill + tiles - 1) / tiles, most = (Sk + kPartKeys - 1) / kPartKeys;
  return {false, want < most ? want : most};
}

size_t part_bytes(const DiffPlan& p, int64_t B, int64_t Hk, int64_t R, int64_t Dv) {
  if (!p.few && p.n_parts <= 1) return 0;
  const size_t rows = size_t(p.n_parts) * size_t(p.few ? 1 : B) * size_t(Hk) * size_t(R) * 2;
  return (rows * size_t(Dv) + rows * 4) * sizeof(float);
}

// Sizes that the kernels' 32-bit row and key numbers and the grids hold. A cache's
// capacity is no part of a grid (the rows say how many parts there are), but FewParts
// counts all of its blocks of 32 keys.
bool sizes_ok(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk, bool cached) {
  if (B < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || Sq < 0 || Sk < 0) return false;
  const int64_t lim = int64_t(1) << 30;
  return B < lim && H < lim && Sq < lim && Sk < lim && tjh::product_below(lim, {Sq, H / Hk}) &&
         tjh::product_below(lim, {Sk, H / Hk}) && tjh::product_below(lim, {B, H}) &&
         tjh::product_below(int64_t(1) << 56, {B, H, Sq + 128, 1024}) && tjh::product_below(int64_t(1) << 35, {B, Sk}) &&
         // workgroups of 256 threads: one for every 128 rows or keys, and up to 512 more in parts
         tjh::product_below(int64_t(1) << 22, {B, Hk, (Sq / 128 + 1) * (H / Hk) + (cached ? 0 : Sk / 128) + 2});
}

int check_dims(int dtype, int64_t D, int64_t Dv) {
  const int elt = elem_bytes(dtype);
  if (elt == 0) return TJ_ERR_DTYPE;
  if (D <= 0 || Dv <= 0) return TJ_ERR_SHAPE;
  if (D > 128 || Dv > 256) return TJ_ERR_UNSUPPORTED;
  if (D * elt % 16 != 0 || Dv * elt % 16 != 0) return TJ_ERR_ALIGN;
  return TJ_OK;
}

bool view_ok(const void* p, const int64_t st[4], int dtype) {
  const int64_t vec = 16 / elem_bytes(dtype);
  if (st == nullptr || st[3] != 1 || !tjh::aligned16(p)) return false;
  return st[0] % vec == 0 && st[1] % vec == 0 && st[2] % vec == 0;
}

// Rows that the tile copies reach by 31-bit byte offsets, up to 64 at a time.
bool rows_ok(const int64_t st[4], int dtype) {
  return st[2] >= 0 && st[2] < (int64_t(1) << 31) / (64 * elem_bytes(dtype));
}

View4 view(const int64_t st[4]) { return View4{st[0], st[1], st[2]}; }

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace
}  // namespace tj

using namespace tj;

extern "C" size_t tj_diff_attn_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk, int64_t Dv,
                                               int cached) {
  if (!sizes_ok(B, H, Hk, Sq, Sk, cached != 0) || Dv <= 0 || Dv > 256 || B == 0 || Sq == 0) return 0;
  const int64_t R = Sq * (H / Hk);
  return part_bytes(plan(B, Hk, R, Sk, Dv, cached != 0), B, Hk, R, Dv);
}

extern "C" int tj_diff_attn_fwd(const void* q, const void* k, const void* v, void* o, int dtype, int64_t B, int64_t H,
                                int64_t Hk, int64_t Sq, int64_t Sk, int64_t D, int64_t Dv, const int64_t q_strides[4],
                                const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
                                float scale, int causal, int cached, const float* lam, int64_t lam_step,
                                const int32_t* lengths, float* lse, float* maps, void* workspace, size_t workspace_bytes,
                                hipStream_t stream) {
  if (elem_bytes(dtype) == 0) return TJ_ERR_DTYPE;
  if (!sizes_ok(B, H, Hk, Sq, Sk, cached != 0)) return TJ_ERR_SHAPE;
  if (const int rc = check_dims(dtype, D, Dv)) return rc;
  if (cached ? lengths == nullptr : Sq != Sk) return TJ_ERR_SHAPE;
  if ((lam_step != 0 && lam_step != 1) || (lse == nullptr) != (maps == nullptr)) return TJ_ERR_SHAPE;
  if (B == 0 || Sq == 0) return TJ_OK;
  if (q == nullptr || o == nullptr || lam == nullptr || (Sk > 0 && (k == nullptr || v == nullptr))) return TJ_ERR_SHAPE;
  if (!view_ok(q, q_strides, dtype) || !view_ok(k, k_strides, dtype) || !view_ok(v, v_strides, dtype) ||
      !view_ok(o, o_strides, dtype) || !tjh::aligned16(maps) || !aligned4(lam) || !aligned4(lengths) || !aligned4(lse))
    return TJ_ERR_ALIGN;
  if (!rows_ok(k_strides, dtype) || !rows_ok(v_strides, dtype)) return TJ_ERR_UNSUPPORTED;
  DiffArgs a{};
  a.q = q; a.k = k; a.v = v; a.o = o; a.maps = maps;
  a.vq = view(q_strides); a.vk = view(k_strides); a.vv = view(v_strides); a.vo = view(o_strides);
  a.B = (int)B; a.H = (int)H; a.Hk = (int)Hk; a.G = (int)(H / Hk); a.D = (int)D; a.Dv = (int)Dv;
  a.Sq = (int)Sq; a.Sk = (int)Sk; a.R = (int)(Sq * a.G);
  a.scale = scale; a.causal = causal != 0 || cached != 0; a.cached = cached != 0;
  a.lam = lam; a.lam_step = (int)lam_step; a.len = lengths; a.lse = lse;
  const DiffPlan p = plan(B, Hk, a.R, Sk, Dv, a.cached);
  const size_t need = part_bytes(p, B, Hk, a.R, Dv);
  // diff_join_kernel: a workgroup per row. (A cache of no capacity still has rows to clear.)
  if ((p.few || need != 0) && B * Hk * a.R >= (int64_t(1) << 24)) return TJ_ERR_SHAPE;
  a.n_parts = 1;
  if (need != 0 && (p.few || workspace != nullptr)) {
    if (workspace == nullptr || workspace_bytes < need) return TJ_ERR_WORKSPACE;
    if (!tjh::aligned16(workspace)) return TJ_ERR_ALIGN;
    a.n_parts = (int)p.n_parts;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + need / sizeof(float) / (Dv + 4) * Dv;
  }
  return p.few ? diff_few_rows(a, dtype, stream) : diff_fwd(a, dtype, stream);
}

extern "C" size_t tj_diff_attn_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t S) {
  if (!sizes_ok(B, H, Hk, S, S, false)) return 0;
  return (size_t(B) * size_t(H) * (size_t(S) * 3 + size_t(stat_rows(S)) * 4) + size_t(B) * size_t(Hk) * 2 * kPeakParts) *
         sizeof(float);
}

extern "C" int tj_diff_attn_bwd(const void* q, const void* k, const void* v, const float* maps, const float* lse,
                                const void* dout, void* dq, void* dk, void* dv, float* dlam, int dtype,
                                int64_t B, int64_t H, int64_t Hk, int64_t S, int64_t D, int64_t Dv,
                                const int64_t q_strides[4], const int64_t k_strides[4], const int64_t v_strides[4],
                                const int64_t do_strides[4], const int64_t dq_strides[4], const int64_t dk_strides[4],
                                const int64_t dv_strides[4], float scale, int causal,
                                const float* lam, int64_t lam_step, const int32_t* lengths, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
  if (elem_bytes(dtype) == 0) return TJ_ERR_DTYPE;
  if (!sizes_ok(B, H, Hk, S, S, false)) return TJ_ERR_SHAPE;
  if (const int rc = check_dims(dtype, D, Dv)) return rc;
  if (lam_step != 0 && lam_step != 1) return TJ_ERR_SHAPE;
  if (lam == nullptr || dlam == nullptr) return TJ_ERR_SHAPE;
  if (B == 0 || S == 0) return TJ_OK;
  for (const void* p : {q, k, v, (const void*)maps, (const void*)lse, dout, (const void*)dq, (const void*)dk, (const void*)dv})
    if (p == nullptr) return TJ_ERR_SHAPE;
  if (!view_ok(q, q_strides, dtype) || !view_ok(k, k_strides, dtype) || !view_ok(v, v_strides, dtype) ||
      !tjh::aligned16(maps) || !view_ok(dout, do_strides, dtype) ||
      !view_ok(dq, dq_strides, dtype) || !view_ok(dk, dk_strides, dtype) || !view_ok(dv, dv_strides, dtype) ||
      !aligned4(lam) || !aligned4(dlam) || !aligned4(lengths) || !aligned4(lse))
    return TJ_ERR_ALIGN;
  for (const int64_t* st : {q_strides, k_strides, v_strides, do_strides})
    if (!rows_ok(st, dtype)) return TJ_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < tj_diff_attn_bwd_workspace_bytes(B, H, Hk, S)) return TJ_ERR_WORKSPACE;
  if (!tjh::aligned16(workspace)) return TJ_ERR_ALIGN;
  DiffArgs a{};
  a.q = q; a.k = k; a.v = v; a.maps = const_cast<float*>(maps);
  a.vq = view(q_strides); a.vk = view(k_strides); a.vv = view(v_strides);
  a.vdo = view(do_strides); a.vdq = view(dq_strides); a.vdk = view(dk_strides); a.vdv = view(dv_strides);
  a.B = (int)B; a.H = (int)H; a.Hk = (int)Hk; a.G = (int)(H / Hk); a.D = (int)D; a.Dv = (int)Dv;
  a.Sq = a.Sk = (int)S; a.R = (int)(S * a.G);
  a.scale = scale; a.causal = causal != 0;
  a.lam = lam; a.lam_step = (int)lam_step; a.len = lengths; a.lse = const_cast<float*>(lse);
  a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv; a.dlam = dlam;
  a.n_lam = lam_step ? (int)H : 1;
  a.delta = static_cast<float*>(workspace);
  a.gsum = a.delta + 2 * B * H * S;
  a.stat = a.gsum + B * H * S;
  a.peak = a.stat + B * H * 4 * stat_rows(S);
  const int64_t blocks = ((int64_t)a.R + 63) / 64;
  a.n_peaks = (int)(blocks < kPeakParts ? blocks : kPeakParts);
  if (const int rc = diff_delta(a, dtype, stream)) return rc;
  // dQ first: it leaves the exact delta for dK.
  if (const int rc = diff_bwd_q(a, dtype, stream)) return rc;
  return diff_bwd_kv(a, dtype, stream);
}
