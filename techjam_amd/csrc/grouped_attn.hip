// Attention with grouped heads, packed sequences and drafted tokens: the C ABI entry
// points and their argument checks. The kernels are in packed_attn_fwd.hip,
// packed_attn_bwd.hip and tree_attn.hip.
#include <algorithm>

#include "grouped_attn.h"

namespace tj {
namespace {

int elem_bytes(int dtype) { return dtype == TJ_F32 ? 4 : (dtype == TJ_F16 || dtype == TJ_BF16 ? 2 : 0); }

int check_dims(int dtype, int64_t D, int64_t Dv) {
  const int elt = elem_bytes(dtype);
  if (elt == 0) return TJ_ERR_DTYPE;
  if (D <= 0 || Dv <= 0) return TJ_ERR_SHAPE;
  if (D > 128 || Dv > 128) return TJ_ERR_UNSUPPORTED;
  if (D * elt % 16 != 0 || Dv * elt % 16 != 0) return TJ_ERR_ALIGN;
  return TJ_OK;
}

// Unit innermost stride, rows and base aligned to 16 bytes; n strides, the last of them the innermost.
bool view_ok(const void* p, const int64_t* st, int n, int dtype) {
  const int64_t vec = 16 / elem_bytes(dtype);
  if (st == nullptr || st[n - 1] != 1 || !tjh::aligned16(p)) return false;
  for (int i = 0; i + 1 < n; ++i)
    if (st[i] % vec != 0) return false;
  return true;
}

// Rows that the tile copies reach by 31-bit byte offsets, up to 64 at a time.
bool rows_ok(int64_t stride, int dtype) { return stride >= 0 && stride < (int64_t(1) << 31) / (64 * elem_bytes(dtype)); }

// The kernels multiply strides as 32-bit numbers, other than a batch's; n strides.
bool near_ok(std::initializer_list<const int64_t*> views, int n) {
  for (const int64_t* st : views)
    for (int i = n - 3; i < n - 1; ++i)
      if (st[i] >= int64_t(1) << 31 || st[i] <= -(int64_t(1) << 31)) return false;
  return true;
}

bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

// Sizes that the kernels' 32-bit row and slot numbers and the grids (workgroups of up to 512
// threads, one for every 32 rows or keys) hold.
bool packed_sizes_ok(int64_t T, int64_t N, int64_t H, int64_t Hk) {
  if (T < 0 || N < 0 || H <= 0 || Hk <= 0 || H % Hk != 0) return false;
  const int64_t lim = int64_t(1) << 30;
  return T < lim && N < lim && H < lim && tjh::product_below(lim, {T + 64, H}) &&
         tjh::product_below(int64_t(1) << 23, {Hk, (T / 32 + 1) * (H / Hk) + N + 4});
}

PackedArgs packed_args(const void* q, const void* k, const void* v, int64_t T, int64_t N, int64_t H, int64_t Hk, int64_t D,
                       int64_t Dv, const int64_t* qs, const int64_t* ks, const int64_t* vs, const int64_t* os, float scale,
                       int causal, const int32_t* offsets, const int32_t* lengths) {
  PackedArgs a{};
  a.q = q; a.k = k; a.v = v;
  a.vq = View3{qs[0], qs[1]}; a.vk = View3{ks[0], ks[1]}; a.vv = View3{vs[0], vs[1]}; a.vo = View3{os[0], os[1]};
  a.T = (int)T; a.N = (int)N; a.H = (int)H; a.Hk = (int)Hk; a.G = (int)(H / Hk); a.by_group = Divisor::of(a.G); a.D = (int)D; a.Dv = (int)Dv;
  a.scale = scale; a.causal = causal != 0; a.off = offsets; a.len = lengths;
  return a;
}

// The numbers of 32 tokens, then the peaks of 64.
size_t stat_floats(int64_t T, int64_t N, int64_t H) { return size_t(region_slots(T, N, 1, 32)) * size_t(H) * 64; }
size_t peak_floats(int64_t T, int64_t N, int64_t Hk) { return size_t(region_slots(T, N, 1, 64)) * size_t(Hk) * 2; }
// Behind them, from a whole 16 bytes on, the sums of shared key tiles, of the type with most of them and the largest dims.
size_t part_first(int64_t T, int64_t N, int64_t H, int64_t Hk) { return (stat_floats(T, N, H) + peak_floats(T, N, Hk) + 3) / 4 * 4; }
size_t part_floats(int64_t T, int64_t N, int64_t H, int64_t Hk) {
  const int shares = std::max(packed_bwd_shares(TJ_F32, T, N, H, Hk), packed_bwd_shares(TJ_BF16, T, N, H, Hk));
  return shares == 1 ? 0 : size_t(shares) * size_t(T) * size_t(Hk) * 256;
}

// A cache's capacity is no part of a grid, but its blocks of 32 keys are counted.
bool tree_sizes_ok(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk) {
  if (B < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || Sq < 0 || Sk < 0) return false;
  const int64_t lim = int64_t(1) << 30;
  // A workgroup for every 32 rows of a sequence (256 threads and fewer) or for every row (joins), and up
  // to 20 a CU in parts.
  return B < lim && H < lim && Sk < lim && tjh::product_below(lim, {Sq, H / Hk}) && tjh::product_below(int64_t(1) << 35, {B, Sk}) &&
         tjh::product_below(int64_t(1) << 22, {B, Hk}) && tjh::product_below((int64_t(1) << 23) - 65536, {B, H, Sq});
}

TreeArgs tree_sizes(int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk, int64_t D, int64_t Dv) {
  TreeArgs a{};
  a.B = (int)B; a.H = (int)H; a.Hk = (int)Hk; a.G = (int)(H / Hk); a.by_group = Divisor::of(a.G); a.D = (int)D; a.Dv = (int)Dv;
  a.Sq = (int)Sq; a.Sk = (int)Sk; a.R = (int)(Sq * a.G);
  return a;
}

size_t part_rows(const TreeArgs& a, const TreePlan& p) { return size_t(p.parts.total) * size_t(a.Hk) * size_t(a.R); }
size_t part_bytes(const TreeArgs& a, const TreePlan& p) {
  return p.whole() ? 0 : (part_rows(a, p) * size_t(a.Dv + 4) + size_t(a.B) * 2) * sizeof(float);
}

}  // namespace
}  // namespace tj

using namespace tj;

extern "C" int tj_packed_attn_fwd(const void* q, const void* k, const void* v, void* o, int dtype, int64_t T, int64_t N,
                                  int64_t H, int64_t Hk, int64_t D, int64_t Dv, const int64_t q_strides[3],
                                  const int64_t k_strides[3], const int64_t v_strides[3], const int64_t o_strides[3],
                                  float scale, int causal, const int32_t* offsets, const int32_t* lengths, float* lse,
                                  void* o_rest, hipStream_t stream) {
  if (elem_bytes(dtype) == 0) return TJ_ERR_DTYPE;
  if (!packed_sizes_ok(T, N, H, Hk)) return TJ_ERR_SHAPE;
  if (const int rc = check_dims(dtype, D, Dv)) return rc;
  if (T == 0) return TJ_OK;
  for (const void* p : {q, k, v, (const void*)o, (const void*)offsets})
    if (p == nullptr) return TJ_ERR_SHAPE;
  if ((o_rest != nullptr) != (lse != nullptr && dtype != TJ_F32)) return TJ_ERR_SHAPE;
  if (!view_ok(q, q_strides, 3, dtype) || !view_ok(k, k_strides, 3, dtype) || !view_ok(v, v_strides, 3, dtype) ||
      !view_ok(o, o_strides, 3, dtype) || !tjh::aligned16(o_rest) || !aligned4(offsets) || !aligned4(lengths) || !aligned4(lse))
    return TJ_ERR_ALIGN;
  if (!rows_ok(k_strides[0], dtype) || !rows_ok(v_strides[0], dtype) ||
      !near_ok({q_strides, k_strides, v_strides, o_strides}, 3))
    return TJ_ERR_UNSUPPORTED;
  PackedArgs a = packed_args(q, k, v, T, N, H, Hk, D, Dv, q_strides, k_strides, v_strides, o_strides, scale, causal, offsets,
                             lengths);
  a.o = o;
  a.lse = lse;
  a.rest = o_rest;
  return packed_fwd(a, dtype, stream);
}

extern "C" size_t tj_packed_attn_bwd_workspace_bytes(int64_t T, int64_t N, int64_t H, int64_t Hk) {
  if (!packed_sizes_ok(T, N, H, Hk)) return 0;
  return (part_first(T, N, H, Hk) + part_floats(T, N, H, Hk)) * sizeof(float);
}

extern "C" int tj_packed_attn_bwd(const void* q, const void* k, const void* v, const void* o,
                                  const void* o_rest, const float* lse, const void* dout, void* dq, void* dk, void* dv, int dtype, int64_t T, int64_t N, int64_t H,
                                  int64_t Hk, int64_t D, int64_t Dv, const int64_t q_strides[3], const int64_t k_strides[3],
                                  const int64_t v_strides[3], const int64_t o_strides[3], const int64_t do_strides[3],
                                  const int64_t dq_strides[3], const int64_t dk_strides[3], const int64_t dv_strides[3],
                                  float scale, int causal, const int32_t* offsets, const int32_t* lengths, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (elem_bytes(dtype) == 0) return TJ_ERR_DTYPE;
  if (!packed_sizes_ok(T, N, H, Hk)) return TJ_ERR_SHAPE;
  if (const int rc = check_dims(dtype, D, Dv)) return rc;
  if (T == 0) return TJ_OK;
  for (const void* p : {q, k, v, o, (const void*)lse, dout, (const void*)dq, (const void*)dk, (const void*)dv,
                        (const void*)offsets})
    if (p == nullptr) return TJ_ERR_SHAPE;
  if ((o_rest != nullptr) != (dtype != TJ_F32)) return TJ_ERR_SHAPE;
  if (!view_ok(q, q_strides, 3, dtype) || !view_ok(k, k_strides, 3, dtype) || !view_ok(v, v_strides, 3, dtype) ||
      !view_ok(o, o_strides, 3, dtype) || !tjh::aligned16(o_rest) || !view_ok(dout, do_strides, 3, dtype) || !view_ok(dq, dq_strides, 3, dtype) ||
      !view_ok(dk, dk_strides, 3, dtype) || !view_ok(dv, dv_strides, 3, dtype) || !aligned4(offsets) || !aligned4(lengths) ||
      !aligned4(lse))
    return TJ_ERR_ALIGN;
  for (const int64_t* st : {q_strides, k_strides, v_strides, do_strides})
    if (!rows_ok(st[0], dtype)) return TJ_ERR_UNSUPPORTED;
  if (!near_ok({q_strides, k_strides, v_strides, o_strides, do_strides, dq_strides, dk_strides, dv_strides}, 3))
    return TJ_ERR_UNSUPPORTED;
  if (workspace == nullptr || workspace_bytes < tj_packed_attn_bwd_workspace_bytes(T, N, H, Hk)) return TJ_ERR_WORKSPACE;
  if (!tjh::aligned16(workspace)) return TJ_ERR_ALIGN;
  PackedArgs a = packed_args(q, k, v, T, N, H, Hk, D, Dv, q_strides, k_strides, v_strides, o_strides, scale, causal, offsets,
                             lengths);
  a.out = o; a.rest = const_cast<void*>(o_rest); a.lse = const_cast<float*>(lse); a.dout = dout;
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.vdo = View3{do_strides[0], do_strides[1]}; a.vdq = View3{dq_strides[0], dq_strides[1]};
  a.vdk = View3{dk_strides[0], dk_strides[1]}; a.vdv = View3{dv_strides[0], dv_strides[1]};
  a.stat = static_cast<float*>(workspace);
  a.peak = a.stat + stat_floats(T, N, H);
  a.shares = packed_bwd_shares(dtype, T, N, H, Hk);
  a.part = a.stat + part_first(T, N, H, Hk);
  return packed_bwd(a, dtype, stream);
}

extern "C" size_t tj_tree_attn_workspace_bytes(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t Sq, int64_t Sk, int64_t D,
                                               int64_t Dv) {
  if (!tree_sizes_ok(B, H, Hk, Sq, Sk) || check_dims(dtype, D, Dv) != TJ_OK || B == 0 || Sq == 0) return 0;
  const TreeArgs a = tree_sizes(B, H, Hk, Sq, Sk, D, Dv);
  return part_bytes(a, tree_plan(a, dtype));
}

extern "C" int tj_tree_attn_fwd(const void* q, const void* k, const void* v, void* o, int dtype, int64_t B, int64_t H,
                                int64_t Hk, int64_t Sq, int64_t Sk, int64_t D, int64_t Dv, const int64_t q_strides[4],
                                const int64_t k_strides[4], const int64_t v_strides[4], const int64_t o_strides[4],
                                float scale, const int32_t* lengths, const int32_t* parents, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
  if (elem_bytes(dtype) == 0) return TJ_ERR_DTYPE;
  if (!tree_sizes_ok(B, H, Hk, Sq, Sk)) return TJ_ERR_SHAPE;
  if (const int rc = check_dims(dtype, D, Dv)) return rc;
  if (parents != nullptr && Sq > 64) return TJ_ERR_UNSUPPORTED;
  if (B == 0 || Sq == 0) return TJ_OK;
  if (q == nullptr || o == nullptr || lengths == nullptr || (Sk > 0 && (k == nullptr || v == nullptr))) return TJ_ERR_SHAPE;
  if (!view_ok(q, q_strides, 4, dtype) || !view_ok(k, k_strides, 4, dtype) || !view_ok(v, v_strides, 4, dtype) ||
      !view_ok(o, o_strides, 4, dtype) || !aligned4(lengths) || !aligned4(parents))
    return TJ_ERR_ALIGN;
  if (!rows_ok(k_strides[2], dtype) || !rows_ok(v_strides[2], dtype) || !near_ok({q_strides, o_strides}, 4))
    return TJ_ERR_UNSUPPORTED;
  TreeArgs a = tree_sizes(B, H, Hk, Sq, Sk, D, Dv);
  a.q = q; a.k = k; a.v = v; a.o = o;
  a.vq = View4{q_strides[0], q_strides[1], q_strides[2]}; a.vk = View4{k_strides[0], k_strides[1], k_strides[2]};
  a.vv = View4{v_strides[0], v_strides[1], v_strides[2]}; a.vo = View4{o_strides[0], o_strides[1], o_strides[2]};
  a.scale = scale; a.len = lengths; a.parents = parents;
  const TreePlan p = tree_plan(a, dtype);
  if (const size_t bytes = part_bytes(a, p)) {
    if (workspace == nullptr || workspace_bytes < bytes) return TJ_ERR_WORKSPACE;
    if (!tjh::aligned16(workspace)) return TJ_ERR_ALIGN;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + part_rows(a, p) * size_t(Dv);
    a.plan = reinterpret_cast<int32_t*>(a.part_ml + part_rows(a, p) * 4);
  }
  return tree_fwd(a, p, dtype, stream);
}
