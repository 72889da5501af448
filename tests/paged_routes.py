"""Calls of mtg_paged_attn_dev by the way the library takes through them: which kernel, how its splits are joined.
test_serve_checks.py holds on the CPU that each call still takes the route that it stands for here, and
test_gpu_paged_attn_routes.py compares its result with the 64-bit form."""

# Route: kernel and join. rows16 / rows32: k_paged_rows with tiles of 16 / 32 (row, head) pairs, rows16x8 with eight
# waves; chunk: k_paged_chunk. alone: no splits; marks: joined in the same launch; join1 / 4 / 16: by a second launch of
# that many waves a row. An f32 cache never takes k_paged_chunk: its route where it differs stands behind the "|".
SHORT = [(1, 50), (0, 9), (1, 700), (1, 33)]
CASES = [
    # name, heads, kv_heads, lens, window, max_kv (0: the longest length), route
    ("one token, one split", 4, 2, [(1, 100), (1, 1), (0, 3)], 0, 0, "rows16 alone"),
    ("one token, few splits", 16, 8, [(1, 613)], 0, 0, "rows16 marks"),
    ("one token, many splits", 2, 1, [(1, 9000), (2, 700)], 0, 0, "rows16 marks"),
    ("many sequences, two splits", 16, 8, [(1, 40 + 61 * i) for i in range(35)] + [(0, 3000), (1, 1), (1, 0)], 0, 2200, "rows16 join1"),
    ("several tokens, a dozen splits", 16, 8, [(4, 8100), *SHORT, (3, 2000)], 0, 0, "rows16 join4"),
    ("long contexts", 8, 8, [(1, 40000), *SHORT], 0, 0, "rows16 join16"),
    ("long contexts, shared heads", 16, 8, [(1, 33000), (2, 20000), *SHORT[:2]], 0, 0, "rows16 join16"),
    ("a long context's window", 8, 8, [(1, 40000), (1, 36000), *SHORT], 34000, 0, "rows16 join16"),
    ("longer than was expected", 8, 8, [(1, 40000), *SHORT], 0, 35000, "rows16 join16"),
    ("short contexts", 16, 8, [(1, 1 + 40 * i) for i in range(16)], 0, 640, "rows16x8 alone"),
    ("drafts, one split", 4, 2, [(9, 100), (10, 12), (9, 9)], 0, 0, "rows32 alone"),
    ("drafts, few splits", 4, 2, [(9, 1500), (10, 700)], 0, 0, "rows32 marks"),
    ("drafts, two splits", 4, 2, [(9, 40 + 61 * i) for i in range(35)] + [(0, 3000), (9, 9), (9, 0)], 0, 2200, "rows32 join1"),
    ("drafts, a dozen splits", 8, 8, [(17, 12000), (20, 600), (18, 9000)], 0, 0, "rows32 join4"),
    ("drafts, long contexts", 8, 8, [(17, 17300)], 0, 0, "rows32 join16"),
    ("drafts, a long context's window", 8, 8, [(17, 20000)], 17200, 0, "rows32 join16"),
    ("a chunk, one split", 4, 2, [(70, 100), (90, 91)], 0, 0, "chunk alone|rows32 alone"),
    ("a chunk, few splits", 4, 2, [(150, 1900), (90, 95), (70, 700)], 0, 0, "chunk join1|rows32 marks"),
    ("a chunk, a dozen splits", 2, 1, [(100, 4000), (40, 60)], 0, 0, "chunk join4|rows32 marks"),
    ("a chunk, long context", 1, 1, [(100, 9500)], 0, 0, "chunk join16|rows32 marks"),
    ("a chunk, long context's window", 2, 1, [(60, 14000)], 10000, 0, "chunk join16|rows32 marks"),
    ("a chunk and a token, long contexts", 1, 1, [(150, 12000), (1, 11000)], 0, 0, "chunk join16|rows32 marks"),
]
PAGE = 64


def table_stride(lens):
    """Of serve_ref.Batch."""
    return max([-(-max(0, length) // PAGE) for _, length in lens] + [1]) + 1


def call(case, io, kv, dim):
    """The call as tests/cpp/test_serve_calls.cpp reads it."""
    _, heads, kv_heads, lens, window, max_kv, _ = case
    return (int(io[1:]), int(kv[1:]), heads, kv_heads, dim, PAGE, len(lens), sum(n for n, _ in lens), table_stride(lens), window,
            max_kv or max(length for _, length in lens))


def route(case, kv):
    both = case[-1].split("|")
    return both[-1] if kv == "f32" else both[0]
