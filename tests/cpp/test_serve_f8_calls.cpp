// The host code of the operators over a cache in 8 bits and of the sampler on the fake HIP runtime. For each line of standard
// input, an attention call,
//   io heads kv_heads head_dim page_size n_seqs n_tokens table_stride window sink max_kv     (io: 16 or 32 bits)
// a line with its workspace in bytes and the kernels it launches, by their mangled names, each with its dynamic LDS, or "refused".
#include "fake_hip.hpp"

#include <cstdio>

#include "mtg_verify.h"

static int failures = 0;
static void expect(bool ok, const char* what) {
  if (ok) return;
  std::fprintf(stderr, "FAILED: %s: %s\n", what, mtg_last_error(nullptr));
  ++failures;
}
// Addresses that nothing reads: the fake runtime runs no kernel.
static void* at(uint64_t gigabytes) { return (void*)((1ull << 40) + (gigabytes << 30)); }

static mtg_paged_kv cache(int kv_heads, int dim, int page, int n_seqs, int n_tokens, int table_stride) {
  mtg_paged_kv c{};
  c.k = at(0), c.v = at(100);
  c.page_table = (const int32_t*)at(200), c.kv_len = (const int32_t*)at(201), c.q_start = (const int32_t*)at(202);
  c.head_stride = (int64_t)page * dim;
  c.page_stride = c.head_stride * kv_heads;
  c.kv_type = MTG_TYPE_F8_E4M3;
  c.n_pages = 4, c.page_size = page, c.table_stride = table_stride;
  c.n_seqs = n_seqs, c.n_tokens = n_tokens, c.n_kv_heads = kv_heads, c.head_dim = dim;
  return c;
}
static mtg_f8_scales scales(int kv_heads, int page) {
  mtg_f8_scales s{};
  s.k = (uint8_t*)at(250), s.v = (uint8_t*)at(260);
  s.head_stride = page / MTG_F8_BLOCK, s.page_stride = s.head_stride * kv_heads;
  return s;
}

static void routes() {
  int io, heads, kv_heads, dim, page, n_seqs, n_tokens, table_stride, window, sink, max_kv;
  while (std::scanf("%d %d %d %d %d %d %d %d %d %d %d", &io, &heads, &kv_heads, &dim, &page, &n_seqs, &n_tokens, &table_stride, &window,
                    &sink, &max_kv) == 11) {
    mtg_paged_attn_f8 x{};
    mtg_paged_attn& a = x.a;
    a.kv = cache(kv_heads, dim, page, n_seqs, n_tokens, table_stride);
    x.scales = scales(kv_heads, page), x.sink = sink;
    a.q = at(300), a.out = at(400), a.q_stride = a.out_stride = (int64_t)heads * dim;
    a.io_type = io == 16 ? MTG_TYPE_F16 : MTG_TYPE_F32;
    a.n_heads = heads, a.window = window, a.max_kv = max_kv, a.scale = 0.1f;
    a.workspace_bytes = mtg_paged_attn_f8_workspace(&x);
    a.workspace = at(500);
    fake::state().launches.clear();
    if (mtg_paged_attn_f8_dev(&x, nullptr) != MTG_OK) {
      std::printf("refused\n");
      continue;
    }
    std::printf("%zu", a.workspace_bytes);
    for (const fake::Launch& l : fake::state().launches) std::printf(" %s %zu", l.kernel.c_str(), l.lds);
    std::printf("\n");
  }
}

// Launches of a call, all on its stream.
static int launched(int rc, void* stream) {
  int n = 0;
  for (const fake::Launch& l : fake::state().launches) n += l.stream == stream;
  const bool all = n == (int)fake::state().launches.size();
  fake::state().launches.clear();
  return rc == MTG_OK && all ? n : -1;
}

static void others() {
  fake::state().launches.clear();
  void* stream = at(900);
  for (int rows : {1, 4, 5, 300, 20000}) {
    mtg_rope_append_f8 x{};
    x.a.kv = cache(8, 128, 64, 1, rows, 400);
    x.scales = scales(8, 64);
    x.a.q = at(300), x.a.k_new = at(310), x.a.v_new = at(320), x.a.q_out = at(330), x.a.freqs = (const double*)at(340);
    x.a.q_stride = x.a.q_out_stride = 2048, x.a.k_stride = x.a.v_stride = 1024;
    x.a.io_type = MTG_TYPE_F16, x.a.n_heads = 16, x.a.rot_dim = 128, x.a.mscale = 1.0f;
    expect(launched(mtg_rope_append_f8_dev(&x, stream), stream) == 1, "append");
  }
  for (int vocab : {1, 1024, 1025, 151936}) {
    mtg_sample s{};
    s.logits = at(0), s.stride = vocab, s.settings = (const float*)at(10), s.uniform = (const float*)at(11), s.choice = (int32_t*)at(12);
    s.io_type = MTG_TYPE_F32, s.rows = 3, s.vocab = vocab;
    s.workspace_bytes = mtg_sample_workspace(&s), s.workspace = at(20);
    expect(launched(mtg_sample_dev(&s, stream), stream) == (vocab > 1024 ? 4 : 2), "sample");
  }
}

int main() {
  routes();
  others();
  std::printf("{\"record\": \"serveF8Calls\", \"failures\": %d}\n", failures);
  return failures != 0;
}
