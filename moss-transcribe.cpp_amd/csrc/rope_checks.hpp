// rope_checks.hpp - what the calls that append rows to a paged cache refuse.
#pragma once

#include "paged_kv.hpp"

namespace mtg {
namespace rope {

// Why the call cannot be made, or nullptr (also where it has nothing to do); *rc gets the status. f8: the cache is held
// in 8 bits, with these scales.
inline const char* refused(const mtg_rope_append& a, bool f8, int* rc, const mtg_f8_scales* scales = nullptr) {
  using namespace paged;
  const mtg_paged_kv& kv = a.kv;
  auto no = [&](int status, const char* why) {
    *rc = status;
    return why;
  };
  const bool with_q = a.q || a.q_out, with_kv = a.k_new || a.v_new;
  if (const char* why = check(kv, with_kv, rc, f8)) return why;
  if (f8 && a.io_type != MTG_TYPE_F32 && a.io_type != MTG_TYPE_F16) return no(MTG_ERR_UNSUPPORTED, "types: rows are f32 or f16");
  if (!f8 && !(a.io_type == MTG_TYPE_F32 && (!with_kv || kv.kv_type == MTG_TYPE_F32 || kv.kv_type == MTG_TYPE_F16)) &&
      !(a.io_type == MTG_TYPE_F16 && (!with_kv || kv.kv_type == MTG_TYPE_F16)))
    return no(MTG_ERR_UNSUPPORTED, "types: f32 rows with an f32 or f16 cache, f16 rows with an f16 cache");
  if (a.rot_dim < 0 || a.rot_dim > kv.head_dim || a.rot_dim % 2) return no(MTG_ERR_INVALID, "rot_dim");
  if (with_q && (a.n_heads <= 0 || a.n_heads > 1024)) return no(MTG_ERR_INVALID, "n_heads");
  if ((a.q == nullptr) != (a.q_out == nullptr)) return no(MTG_ERR_INVALID, "one of q and q_out is NULL");
  if ((a.k_new == nullptr) != (a.v_new == nullptr)) return no(MTG_ERR_INVALID, "one of k_new and v_new is NULL");
  if (kv.n_seqs == 0 || kv.n_tokens == 0) return nullptr;
  if (!with_q && !with_kv) return no(MTG_ERR_INVALID, "neither q nor k and v");
  if (a.rot_dim && !a.freqs) return no(MTG_ERR_INVALID, "freqs is NULL");
  if (!aligned(a.freqs, 8) || !aligned(a.positions, 4)) return no(MTG_ERR_INVALID, "unaligned freqs or positions");
  if (!aligned(a.q_norm, 16) || !aligned(a.k_norm, 16))
    return no(MTG_ERR_UNSUPPORTED, "norms not aligned to 16 bytes");
  const int64_t unit = 16 / (int64_t)type_bytes(a.io_type);
  const int64_t qw = with_q ? (int64_t)a.n_heads * kv.head_dim : 0, kw = with_kv ? (int64_t)kv.n_kv_heads * kv.head_dim : 0;
  const struct {
    const void* at;
    int64_t stride, width;
  } in[] = {{a.q, a.q_stride, qw}, {a.k_new, a.k_stride, kw}, {a.v_new, a.v_stride, kw}, {a.q_out, a.q_out_stride, qw}};
  for (const auto& x : in) {
    if (!x.at) continue;
    if (x.stride < x.width || x.stride > ((int64_t)1 << 40) || !reaches(kv.n_tokens, x.stride))
      return no(MTG_ERR_INVALID, "a row stride below the row's width, or rows behind 2^46 elements");
    if (!aligned(x.at, 16) || x.stride % unit) return no(MTG_ERR_UNSUPPORTED, "rows not aligned to 16 bytes");
  }
  const size_t eb = type_bytes(a.io_type), out_bytes = extent(kv.n_tokens, a.q_out_stride, qw, eb);
  // rows that interleave with another operand's (slices of one wide product) share no element
  // only if the strides are one and the columns apart; that is what in place means here
  auto apart = [&](const void* x, int64_t stride, int64_t width) {
    if (!overlap(a.q_out, out_bytes, x, extent(kv.n_tokens, stride, width, eb))) return true;
    if (stride != a.q_out_stride) return false;
    const int64_t row = stride * (int64_t)eb;
    const int64_t gap = (((int64_t)((uintptr_t)x - (uintptr_t)a.q_out)) % row + row) % row;
    return gap >= qw * (int64_t)eb && gap + width * (int64_t)eb <= row;
  };
  if (with_q) {
    if (!(a.q == a.q_out && a.q_stride == a.q_out_stride) && !apart(a.q, a.q_stride, qw))
      return no(MTG_ERR_INVALID, "q_out overlaps q");
    if (with_kv && (!apart(a.k_new, a.k_stride, kw) || !apart(a.v_new, a.v_stride, kw)))
      return no(MTG_ERR_INVALID, "q_out overlaps k_new or v_new");
  }
  // the other arrays that are read; what one workgroup writes others may still read
  auto shared = [&](const void* p, size_t n) {
    return meets(p, n, {{a.positions, 4 * (size_t)kv.n_tokens}, {a.freqs, 4 * (size_t)a.rot_dim},
                        {a.q_norm, with_q ? 4 * (size_t)kv.head_dim : 0}, {a.k_norm, with_kv ? 4 * (size_t)kv.head_dim : 0},
                        {kv.page_table, with_kv ? 4 * (size_t)kv.n_seqs * kv.table_stride : 0},
                        {kv.kv_len, 4 * (size_t)kv.n_seqs}, {kv.q_start, 4 * (size_t)kv.n_seqs + 4}});
  };
  if (with_q && shared(a.q_out, out_bytes)) return no(MTG_ERR_INVALID, "q_out overlaps an index array, the frequencies or a norm");
  if (with_kv) {
    const size_t pool = pool_extent(kv);
    if (!k_and_v_apart(kv)) return no(MTG_ERR_INVALID, "k and v share elements of one pool");
    for (const void* pages : {kv.k, kv.v}) {
      if (overlap(pages, pool, a.q_out, out_bytes)) return no(MTG_ERR_INVALID, "q_out lies in the pages");
      if (meets(pages, pool, {{a.q, extent(kv.n_tokens, a.q_stride, qw, eb)}, {a.k_new, extent(kv.n_tokens, a.k_stride, kw, eb)},
                              {a.v_new, extent(kv.n_tokens, a.v_stride, kw, eb)}}))
        return no(MTG_ERR_INVALID, "q, k_new or v_new lies in the pages");
      if (shared(pages, pool)) return no(MTG_ERR_INVALID, "an index array, the frequencies or a norm lies in the pages");
    }
  }
  if (f8 && with_kv) {
    if (const char* why = check_scales(kv, *scales, true)) return no(MTG_ERR_INVALID, why);
    const size_t n = scale_extent(kv, *scales);
    for (const uint8_t* x : {scales->k, scales->v})
      if (shared(x, n) || meets(x, n, {{a.q, extent(kv.n_tokens, a.q_stride, qw, eb)}, {a.k_new, extent(kv.n_tokens, a.k_stride, kw, eb)},
                                       {a.v_new, extent(kv.n_tokens, a.v_stride, kw, eb)}, {a.q_out, out_bytes}}))
        return no(MTG_ERR_INVALID, "scales overlap another array");
  }
  return nullptr;
}

}  // namespace rope
}  // namespace mtg
