// The serving operators' host code on the fake HIP runtime. For each line of standard input, a paged attention call,
//   io kv heads kv_heads head_dim page_size n_seqs n_tokens table_stride window max_kv     (io, kv: 16 or 32 bits)
// a line with its workspace in bytes and the kernels it launches, by their mangled names, or "refused".
// Then what calls may look like although arrays meet, on no input: descriptions that are not refused.
#include "fake_hip.hpp"

#include <cstdio>
#include <vector>

#include "mtg_verify.h"

static int failures = 0;
static void expect(bool ok, const char* what) {
  if (ok) return;
  std::fprintf(stderr, "FAILED: %s: %s\n", what, mtg_last_error(nullptr));
  ++failures;
}
// Addresses that nothing reads: the fake runtime runs no kernel.
static void* at(uint64_t gigabytes, uint64_t bytes = 0) { return (void*)((1ull << 40) + (gigabytes << 30) + bytes); }

static mtg_paged_kv cache(int kv, int kv_heads, int dim, int page, int n_seqs, int n_tokens, int table_stride) {
  mtg_paged_kv c{};
  c.k = at(0), c.v = at(100);
  c.page_table = (const int32_t*)at(200), c.kv_len = (const int32_t*)at(201), c.q_start = (const int32_t*)at(202);
  c.head_stride = (int64_t)page * dim;
  c.page_stride = c.head_stride * kv_heads;
  c.kv_type = kv == 16 ? MTG_TYPE_F16 : MTG_TYPE_F32;
  c.n_pages = 4, c.page_size = page, c.table_stride = table_stride;
  c.n_seqs = n_seqs, c.n_tokens = n_tokens, c.n_kv_heads = kv_heads, c.head_dim = dim;
  return c;
}

static void routes() {
  int io, kv, heads, kv_heads, dim, page, n_seqs, n_tokens, table_stride, window, max_kv;
  while (std::scanf("%d %d %d %d %d %d %d %d %d %d %d", &io, &kv, &heads, &kv_heads, &dim, &page, &n_seqs, &n_tokens, &table_stride,
                    &window, &max_kv) == 11) {
    mtg_paged_attn a{};
    a.kv = cache(kv, kv_heads, dim, page, n_seqs, n_tokens, table_stride);
    a.q = at(300), a.out = at(400), a.q_stride = a.out_stride = (int64_t)heads * dim;
    a.io_type = io == 16 ? MTG_TYPE_F16 : MTG_TYPE_F32;
    a.n_heads = heads, a.window = window, a.max_kv = max_kv, a.scale = 0.1f;
    a.workspace_bytes = mtg_paged_attn_workspace(&a);
    a.workspace = at(500);
    fake::state().launches.clear();
    if (mtg_paged_attn_dev(&a, nullptr) != MTG_OK) {
      std::printf("refused\n");
      continue;
    }
    std::printf("%zu", a.workspace_bytes);
    for (const fake::Launch& l : fake::state().launches) std::printf(" %s", l.kernel.c_str());
    std::printf("\n");
  }
}

static int launched(int rc) {
  const int n = (int)fake::state().launches.size();
  fake::state().launches.clear();
  return rc == MTG_OK ? n : -1;
}

// Arrays side by side without a byte between them, in place, slices of one product; arrays that are not read anywhere.
static void accepted() {
  fake::state().launches.clear();
  mtg_logits_step s{};
  s.rows = 3, s.vocab = 5000, s.stride = s.out_stride = 5000, s.io_type = MTG_TYPE_F32;
  s.n_history = 50, s.n_bias = 70, s.mask_stride = 160;
  uint64_t p = 0;
  auto next = [&](uint64_t bytes) { return p += bytes, at(0, p - bytes); };
  s.workspace = next(96), s.workspace_bytes = 96;
  s.logits = next(60000), s.out = next(60000), s.choice = (int32_t*)next(12), s.history = (const int32_t*)next(200);
  s.hist_range = (const int32_t*)next(24), s.penalties = (const float*)next(36), s.bias_ids = (const int32_t*)next(280);
  s.bias = (const float*)next(280), s.bias_range = (const int32_t*)next(24), s.mask = (const uint32_t*)next(4 * (2 * 160 + 157));
  expect(mtg_logits_step_workspace(&s) == 96 && launched(mtg_logits_step_dev(&s, nullptr)) == 1, "logits side by side");
  s.out = (void*)s.logits;
  expect(launched(mtg_logits_step_dev(&s, nullptr)) == 1, "logits in place");
  s.mask = (const uint32_t*)s.choice, s.choice = nullptr;
  expect(launched(mtg_logits_step_dev(&s, nullptr)) == 1, "without a choice");
  s.history = nullptr, s.hist_range = (const int32_t*)s.out, s.bias = nullptr, s.bias_range = (const int32_t*)s.out;
  expect(launched(mtg_logits_step_dev(&s, nullptr)) == 1, "ranges without lists");

  mtg_rope_append r{};
  r.kv = cache(16, 8, 128, 16, 2, 4, 5);
  r.q = at(300), r.k_new = at(300, 4 * 2048), r.v_new = at(300, 4 * 24 * 128), r.q_out = at(300), r.freqs = (const double*)at(301);
  r.q_stride = r.k_stride = r.v_stride = r.q_out_stride = 4096;
  r.io_type = MTG_TYPE_F32, r.n_heads = 16, r.rot_dim = 128;
  expect(launched(mtg_rope_append_dev(&r, nullptr)) == 1, "q in place in a product");
  mtg_rope_append x = r;
  x.q = x.q_out = nullptr, x.q_norm = (const float*)r.kv.k;
  expect(launched(mtg_rope_append_dev(&x, nullptr)) == 1, "k and v alone, q's norm anywhere");
  x = r;
  x.k_new = x.v_new = nullptr, x.k_norm = (const float*)r.q_out, x.kv.page_table = (const int32_t*)r.q_out, x.kv.k = r.q_out;
  expect(launched(mtg_rope_append_dev(&x, nullptr)) == 1, "q alone, k's norm and the cache anywhere");
  x = r;
  x.rot_dim = 0, x.freqs = (const double*)r.q_out;
  expect(launched(mtg_rope_append_dev(&x, nullptr)) == 1, "no rotation, frequencies anywhere");
  x = r;
  const uint64_t pool = 2 * 4 * 8 * 16 * 128;
  x.kv.v = at(0, pool), x.kv.page_table = (const int32_t*)at(0, 2 * pool), x.kv.kv_len = (const int32_t*)at(0, 2 * pool + 40);
  x.kv.q_start = (const int32_t*)at(0, 2 * pool + 48), x.positions = (const int32_t*)at(0, 2 * pool + 60);
  x.freqs = (const double*)at(0, 2 * pool + 80), x.q_norm = (const float*)at(0, 2 * pool + 592), x.k_norm = x.q_norm;
  x.q = x.q_out = at(0, 2 * pool + 1104), x.k_new = (char*)x.q + 4 * 2048, x.v_new = (char*)x.q + 4 * 24 * 128;
  expect(launched(mtg_rope_append_dev(&x, nullptr)) == 1, "all side by side");

  mtg_paged_attn a{};
  a.kv = cache(16, 8, 128, 16, 2, 4, 5);
  const uint64_t out = 4 * 4 * 2048;
  a.q = a.out = at(300), a.q_stride = a.out_stride = 2048, a.io_type = MTG_TYPE_F32, a.n_heads = 16, a.scale = 0.1f;
  a.kv.page_table = (const int32_t*)at(300, out), a.kv.kv_len = (const int32_t*)at(300, out + 40), a.kv.q_start = (const int32_t*)at(300, out + 48);
  expect(launched(mtg_paged_attn_dev(&a, nullptr)) == 1, "index arrays behind out");
  a.workspace = a.out;
  expect(launched(mtg_paged_attn_dev(&a, nullptr)) == 1, "a workspace that is not needed");
  a.scale = 2.3e38f;
  expect(launched(mtg_paged_attn_dev(&a, nullptr)) == 1, "a large scale");
  a.scale = 0.1f, a.q_stride = a.out_stride = (int64_t)1 << 40, a.kv.page_table = (const int32_t*)at(200), a.kv.kv_len = (const int32_t*)at(201);
  a.kv.q_start = (const int32_t*)at(202), a.q = a.out = (void*)(1ull << 50);
  expect(launched(mtg_paged_attn_dev(&a, nullptr)) == 1, "rows far apart");
}

int main() {
  routes();
  accepted();
  std::printf("{\"record\": \"serveCalls\", \"failures\": %d}\n", failures);
  return failures != 0;
}
