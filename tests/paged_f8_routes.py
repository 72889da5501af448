"""Calls of mtg_paged_attn_f8_dev by the way the library takes through them, in the words of paged_routes.py: which kernel, how
its splits are joined. wide: k_paged_chunk_f8 of eight waves. test_serve_f8_routes.py holds on the CPU that each call still takes the
route that it stands for here, and test_gpu_paged_attn_f8_routes.py compares its result with the 64-bit form."""
import paged_routes

# The calls over an f16 cache, where codes have the same route or the one given here; window and first positions beside it.
OTHER = {"several tokens, a dozen splits": "rows16 marks"}
CASES = [(n, h, k, lens, w, 0, m, OTHER.get(n, r.split("|")[0])) for n, h, k, lens, w, m, r in paged_routes.CASES]
CASES += [
    # name, heads, kv_heads, lens, window, sink, max_kv (0: the longest length), route
    ("a window and first positions", 8, 2, [(1, 30000), (1, 900), (1, 2000)], 2048, 4, 0, "rows16 marks"),
    ("drafts, a window and first positions", 8, 1, [(3, 9000), (4, 900)], 4000, 100, 0, "rows32 marks"),
    ("eight rows a head, many workgroups", 16, 4, [(2, 2900), (2, 1700)] * 16, 0, 0, 0, "rows16 marks"),
    ("sixteen rows a head, a dozen splits", 16, 8, [(8, 8100), (8, 700), (9, 2000), (7, 7)], 0, 0, 0, "rows16 join4"),
    ("a third workgroup on few CUs", 16, 8, [(8, 2400 - 300 * i) for i in range(8)], 0, 0, 5000, "rows16 join1"),
    ("a wide chunk, one split", 7, 1, [(150, 200), (147, 160)], 0, 0, 0, "wide alone"),
    ("a wide chunk, few splits", 7, 1, [(150, 1900), (150, 700)], 0, 0, 0, "wide join1"),
    ("a wide chunk, many splits", 16, 1, [(64, 5000)], 0, 0, 0, "wide join4"),
    ("a wide chunk, long context", 16, 1, [(64, 9500)], 0, 0, 0, "wide join16"),
    ("a wide chunk, a window and first positions", 16, 1, [(70, 20000), (64, 800)], 6000, 70, 0, "wide join4"),
]
PAGE = paged_routes.PAGE


def call(case, io, dim):
    """The call as tests/cpp/test_serve_f8_calls.cpp reads it."""
    _, heads, kv_heads, lens, window, sink, max_kv, _ = case
    return (int(io[1:]), heads, kv_heads, dim, PAGE, len(lens), sum(n for n, _ in lens), paged_routes.table_stride(lens), window, sink,
            max_kv or max(length for _, length in lens))
