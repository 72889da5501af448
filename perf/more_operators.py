"""Operators of a serving program whose cache is held in 8 bits, and the sampler, as measurable cases.

A program that holds many long recordings at once keeps their keys and values in 8 bits: e4m3 codes in the
pages of a pool and one power of two for each block of 16 positions and kv head. A step runs

  append   mtg_rope_append_f8_dev: rotary positions (and the q / k norms) of the new rows; q goes on, k and v
           become codes in the pages, in the scale of their block
  attend   mtg_paged_attn_f8_dev: causal attention of the new rows over those pages; in a long stream over a
           window and the first few positions, which stay visible
  sample   mtg_sample_dev: one id per row of logits by temperature, top-k, top-p and min-p from given random numbers

Sizes are this library's own decoder (16 / 8 heads of 128, 151,936 ids), its contexts and verify widths, and
other head layouts of the same range. Sequences of a batch have different lengths.

With `own` false, run() computes the operators from elementary torch operations, in 32 bits, and in 64 bits
where angles of far positions or values next to a border need them.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16}
BYTES = {"f32": 4, "f16": 2}
CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 16        # positions of a scale
LARGEST = 448.0   # of e4m3
LEAST = -100      # of a scale's exponent
EPS = 1e-6
ROPE_BASE = 1e6
GOLDEN = 0.6180339887498949


def listed():
    return [
        # one recording, one token at a time: the smallest step there is
        dict(name="attend_1x1_877", kind="attend", io="f32", heads=16, kv_heads=8, dim=128, page=16, seqs=1, new=1, ctx=877,
             window=0, sink=0),
        # a batch of recordings of all ages, one token each
        dict(name="attend_32x1_12000", kind="attend", io="f16", heads=16, kv_heads=8, dim=128, page=32, seqs=32, new=1,
             ctx=12000, window=0, sink=0),
        # seven drafts and their seed for each of eight recordings, f32 rows
        dict(name="attend_8x8_5000_f32", kind="attend", io="f32", heads=16, kv_heads=8, dim=128, page=64, seqs=8, new=8,
             ctx=5000, window=0, sink=0),
        # live streams that never end: a window and the first four positions, heads of 64, eight to a kv head
        dict(name="attend_64x1_stream", kind="attend", io="f16", heads=32, kv_heads=4, dim=64, page=16, seqs=64, new=1,
             ctx=30000, window=2048, sink=4),
        # a block of a long prompt, ragged, f32 rows
        dict(name="attend_1x1009_7963", kind="attend", io="f32", heads=16, kv_heads=8, dim=128, page=64, seqs=1, new=1009,
             ctx=7963, window=0, sink=0),
        # blocks of two long prompts, a wide model's heads
        dict(name="attend_2x2048_16384", kind="attend", io="f16", heads=32, kv_heads=8, dim=128, page=64, seqs=2, new=2048,
             ctx=16384, window=0, sink=0),
        # one new row of the library's decoder: norms, half pairs, inside a block that has rows already
        dict(name="append_1x1", kind="append", io="f32", heads=16, kv_heads=8, dim=128, page=16, seqs=1, new=1, ctx=613,
             rot=128, inter=False, factor=1.0, norm=True),
        # interleaved pairs on half of the head, a context stretched eight times, far positions, f32 rows
        dict(name="append_48x13_far", kind="append", io="f32", heads=24, kv_heads=4, dim=128, page=32, seqs=48, new=13,
             ctx=2000, rot=64, inter=True, factor=8.0, norm=False),
        # the rows of a whole long prompt
        dict(name="append_1x16384", kind="append", io="f16", heads=16, kv_heads=8, dim=128, page=64, seqs=1, new=16384, ctx=0,
             rot=128, inter=False, factor=1.0, norm=True),
        # the one row of a sampled step, the usual settings
        dict(name="sample_1", kind="sample", io="f32", rows=1, vocab=151936, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0),
        # verify rows in f16, an odd vocabulary, top-p and min-p without top-k
        dict(name="sample_61_f16", kind="sample", io="f16", rows=61, vocab=151643, temperature=1.2, top_k=0, top_p=0.9,
             min_p=0.02),
        # a large batch of requests with settings of their own, all filters
        dict(name="sample_256", kind="sample", io="f32", rows=256, vocab=151936, temperature=0.9, top_k=200, top_p=0.95,
             min_p=0.01),
    ]


def draw(rng):
    """A case of the same ranges. What costs more than the largest listed case of its kind is drawn again."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = {k: [max(work(c)[w] for c in listed() if c["kind"] == k) for w in ("bytes", "flops")]
            for k in ("attend", "append", "sample")}
    while True:
        kind = rng.choice(["attend", "attend", "append", "sample"])
        if kind == "sample":
            case = dict(kind=kind, io=rng.choice(["f32", "f16"]), rows=log_int(1, 256), vocab=log_int(1000, 151936),
                        temperature=rng.choice([1.0, round(rng.uniform(0.3, 1.7), 2)]), top_k=rng.choice([0, log_int(1, 1000)]),
                        top_p=rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), min_p=rng.choice([0.0, round(rng.uniform(0.001, 0.2), 4)]))
        else:
            kv_heads = rng.choice([1, 2, 4, 8])
            case = dict(kind=kind, io=rng.choice(["f32", "f16"]), heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads,
                        dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]), seqs=log_int(1, 64),
                        new=rng.choice([1, log_int(2, 16), log_int(17, 2048)]), ctx=log_int(1, 32768))
            if kind == "attend":
                case["window"] = rng.choice([0, 0, log_int(16, 8192)])
                case["sink"] = rng.choice([0, log_int(1, 64)]) if case["window"] else 0
            else:
                case.update(rot=rng.choice([case["dim"], case["dim"] // 2, 2 * log_int(4, case["dim"] // 2)]),
                            inter=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 16.0]), norm=rng.random() < 0.5)
        w = work(case)
        if w["bytes"] <= most[kind][0] and w["flops"] <= max(most[kind][1], 1) and pool_bytes(case) < 3 << 30 and padded(case) < 3 << 30:
            return case


# ------------------------------------------------------------------- sizes --
def lengths(case):
    """[(new rows, length of the cache with them)] of each sequence: the first has the full sizes, the others
    1/8 to all of the context and half to all of the new rows."""
    out = []
    for b in range(case["seqs"]):
        u = (b * GOLDEN) % 1.0
        n = case["new"] if b == 0 else max(1, int(round(case["new"] * (1.0 - 0.5 * u))))
        c = case["ctx"] if b == 0 else int(round(case["ctx"] * (0.125 + 0.875 * ((b * GOLDEN * GOLDEN) % 1.0))))
        out.append((n, n + c))
    return out


def pages_of(case):
    return [-(-length // case["page"]) for _, length in lengths(case)]


def pool_bytes(case):
    return 0 if case["kind"] == "sample" else 2 * (sum(pages_of(case)) + 3) * case["page"] * case["kv_heads"] * case["dim"]


def padded(case):
    """Scores of the plain form, which takes all sequences as long as the longest."""
    if case["kind"] != "attend":
        return 0
    return case["seqs"] * case["heads"] * case["new"] * max(length for _, length in lengths(case))


def work(case):
    """Each input read once, each output written once."""
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * BYTES[case["io"]] + 28), "flops": 4 * case["rows"] * case["vocab"]}
    io, d, g = BYTES[case["io"]], case["dim"], case["kv_heads"]
    rows = sum(n for n, _ in lengths(case))
    if case["kind"] == "append":
        blocks = sum((length - 1) // BLOCK - (length - n) // BLOCK + 1 for n, length in lengths(case))
        return {"bytes": rows * d * (io * (2 * case["heads"] + 2 * g) + 2 * g) + 2 * g * blocks,
                "flops": rows * ((case["heads"] + g) * (3 * case["rot"] + 4 * d * case["norm"]) + 2 * 2 * g * d)}
    read, seen = 0, 0
    for n, length in lengths(case):
        first = length - n  # position of the first row
        oldest = max(0, first + 1 - case["window"]) if case["window"] else 0
        read += length - oldest + min(case["sink"], oldest)
        for i in range(n):
            o = max(0, first + i + 1 - case["window"]) if case["window"] else 0
            seen += first + i + 1 - o + min(case["sink"], o)
    return {"bytes": 2 * read * g * d + 2 * read * g // BLOCK + 2 * rows * case["heads"] * d * io,
            "flops": 4 * d * case["heads"] * seen}


# ------------------------------------------------------------------ inputs --
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


class _Draws:
    def __init__(self, seed):
        self.g = torch.Generator(device=_device())
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 31))

    def normal(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g, device=_device(), dtype=torch.float32).to(dtype)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.g, device=_device(), dtype=torch.float32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=_device(), dtype=torch.int64).to(torch.int32)

    def ints(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device=_device(), dtype=torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_device())


def frequencies(case):
    """Radians per position of each pair, in 64 bits, and the factor of the rotated values. A stretched
    context keeps the fast pairs, divides the slow ones by `factor` and blends those between."""
    rot, out = case["rot"], []
    ramp = lambda turns: rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(ROPE_BASE))  # noqa: E731
    low, high = max(math.floor(ramp(32)), 0), min(math.ceil(ramp(1)), rot - 1)
    for i in range(rot // 2):
        f = ROPE_BASE ** (-2.0 * i / rot)
        if case["factor"] > 1:
            slow = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)
            f = f / case["factor"] * slow + f * (1.0 - slow)
        out.append(f)
    return out, 0.1 * math.log(case["factor"]) + 1.0 if case["factor"] > 1 else 1.0


def _exponent(top):
    """The least e, LEAST or more, with top <= LARGEST * 2^e: top = m 2^x with m from 1/2 to 1, LARGEST = 7/8 2^9."""
    m, x = torch.frexp(top)
    return torch.where(top > 0, x - 9 + (m > 0.875), LEAST).clamp(min=LEAST).to(torch.int32)


def _cache(case, r):
    """Pages of a pool in no order, the sequences' tables (no row of them is full), their lengths, and in the
    pages what programs stored there: values of a spread that differs from head to head and from block to block."""
    lens, pages = lengths(case), pages_of(case)
    pool = sum(pages) + 3
    order = r.order(pool)
    table = torch.full((len(lens), max(pages) + 1), -1, dtype=torch.int32, device=_device())
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s = dict(lens=lens, starts=starts, table=table, q_start=_ints(starts), kv_len=_ints([length for _, length in lens]))
    g, d, blocks = case["kv_heads"], case["dim"], case["page"] // BLOCK
    for name in "kv":
        x = r.normal(pool, g, blocks, BLOCK, d)
        x *= (0.5 * r.normal(pool, g, blocks, 1, 1) + 0.7 * r.normal(1, g, 1, 1, 1)).exp() * (1.0 if name == "k" else 0.25)
        e = _exponent(x.abs().amax((3, 4)))
        s[name] = torch.ldexp(x, -e[..., None, None]).to(CODES).view(pool, g, case["page"], d)
        s[name + "_scale"] = (e + 127).to(torch.uint8).view(SCALES)
        del x
    return s


def _prepare_attend(case, r):
    s = _cache(case, r)
    # rows as a rotated, normed q has them: unit variance, some heads sharper than others
    sharp = torch.linspace(0.5, 2.5, case["heads"], device=_device()).view(1, -1, 1)
    s["q"] = (r.normal(s["starts"][-1], case["heads"], case["dim"]) * sharp).to(DTYPES[case["io"]])
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    return s


def _prepare_append(case, r):
    s = _cache(case, r)
    wide = case["heads"] + 2 * case["kv_heads"]
    s["qkv"] = (r.normal(s["starts"][-1], wide, case["dim"]) * 1.5).to(DTYPES[case["io"]])
    freqs, s["mscale"] = frequencies(case)
    s["freqs"] = torch.tensor(freqs, dtype=torch.float64, device=_device())
    s["positions"] = None
    if case["factor"] > 1:  # positions of their own: what was evicted or skipped still counts
        s["positions"] = torch.cat([torch.arange(length - n, length) for n, length in s["lens"]]).to(torch.int32).to(_device())
        s["positions"] += r.ints(4096 * int(case["factor"]), s["starts"][-1])
    s["norm"] = [1.0 + 0.1 * r.normal(case["dim"]) for _ in range(2)] if case["norm"] else [None, None]
    return s


def _prepare_sample(case, r):
    rows, vocab = case["rows"], case["vocab"]
    # a bulk that is never said, and a few dozen ids that compete; some rows are sure of themselves, some are not
    x = 2.0 * r.normal(rows, vocab)
    some = r.ints(vocab, rows, 48).long()
    x.scatter_add_(1, some, 12.0 * r.uniform(rows, 48) * (0.5 + r.uniform(rows, 1)))
    s = {"x": x.to(DTYPES[case["io"]])}
    u = r.uniform(rows, 4)
    t = case["temperature"] * (0.75 + 0.5 * u[:, 0])
    if rows >= 8:
        t[::8] = 0.0  # requests that want the likeliest id
    top_p = 1.0 - (1.0 - case["top_p"]) * (0.5 + u[:, 1])
    s["settings"] = torch.stack([t, top_p, case["min_p"] * (0.5 + u[:, 2])], 1).contiguous()
    s["top_k"] = (case["top_k"] * (0.5 + u[:, 3])).ceil().to(torch.int32) if case["top_k"] else None
    s["uniform"] = r.uniform(rows)
    return s


PREPARE = {"attend": _prepare_attend, "append": _prepare_append, "sample": _prepare_sample}


def prepare(case, seed):
    s = PREPARE[case["kind"]](case, _Draws(seed))
    s["case"] = case
    if own:
        _describe(case, s)
    return s


# ------------------------------------------------------- the library's calls --
def _describe(case, s):
    """The call's description and buffers, which a program keeps from step to step."""
    import ctypes
    pkg = os.path.join(ROOT, "moss-transcribe.cpp_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mtg

    L = mtg.lib()
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    types = {"f32": mtg.TYPE_F32, "f16": mtg.TYPE_F16}
    s["stream"] = torch.cuda.current_stream().cuda_stream
    if case["kind"] == "sample":
        s["choice"] = torch.empty(case["rows"], dtype=torch.int32, device=_device())
        s["prob"] = torch.empty(case["rows"], dtype=torch.float32, device=_device())
        a = d = mtg.Sample(logits=at(s["x"]), stride=case["vocab"], settings=at(s["settings"]), top_k=at(s["top_k"]),
                           uniform=at(s["uniform"]), choice=at(s["choice"]), prob=at(s["prob"]), io_type=types[case["io"]],
                           rows=case["rows"], vocab=case["vocab"])
        s["call"], size = L.mtg_sample_dev, L.mtg_sample_workspace(ctypes.byref(d))
    else:
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        width, blocks = (H + 2 * G) * D, case["page"] // BLOCK
        kv = mtg.PagedKv(k=at(s["k"]), v=at(s["v"]), page_table=at(s["table"]), kv_len=at(s["kv_len"]),
                         q_start=at(s["q_start"]), page_stride=G * case["page"] * D, head_stride=case["page"] * D,
                         kv_type=mtg.TYPE_F8_E4M3, n_pages=s["k"].shape[0], page_size=case["page"],
                         table_stride=s["table"].shape[1], n_seqs=case["seqs"], n_tokens=s["starts"][-1], n_kv_heads=G, head_dim=D)
        scales = mtg.F8Scales(k=at(s["k_scale"]), v=at(s["v_scale"]), page_stride=G * blocks, head_stride=blocks)
        if case["kind"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            a = mtg.PagedAttn(kv=kv, q=at(s["q"]), out=at(s["out"]), q_stride=H * D, out_stride=H * D, io_type=types[case["io"]],
                              n_heads=H, max_kv=max(length for _, length in s["lens"]), window=case["window"], scale=s["scale"])
            d = mtg.PagedAttnF8(a=a, scales=scales, sink=case["sink"])
            a, s["call"], size = d.a, L.mtg_paged_attn_f8_dev, L.mtg_paged_attn_f8_workspace(ctypes.byref(d))
        else:
            s["out"] = torch.empty(s["starts"][-1], H, D, dtype=s["qkv"].dtype, device=_device())
            x, b = at(s["qkv"]), BYTES[case["io"]]
            a = mtg.RopeAppend(kv=kv, q=x, k_new=x + H * D * b, v_new=x + (H + G) * D * b, q_out=at(s["out"]),
                               positions=at(s["positions"]), freqs=at(s["freqs"]), q_norm=at(s["norm"][0]),
                               k_norm=at(s["norm"][1]), q_stride=width, k_stride=width, v_stride=width, q_out_stride=H * D,
                               io_type=types[case["io"]], n_heads=H, rot_dim=case["rot"], interleaved=int(case["inter"]), eps=EPS,
                               mscale=s["mscale"])
            d = mtg.RopeAppendF8(a=a, scales=scales)
            s["call"], size = L.mtg_rope_append_f8_dev, 0
    if size:
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device=_device())
        a.workspace, a.workspace_bytes = at(s["workspace"]), size
    s["desc"], s["arg"] = d, ctypes.byref(d)


def _run_own(s):
    rc = s["call"](s["arg"], s["stream"])
    if rc:
        raise RuntimeError("status %d" % rc)


# ------------------------------------------------------------- plain forms --
def _at(codes):
    return codes.view(torch.uint8)  # bytes can be indexed


def _rows(s):
    """[sequence][new row, as many as the longest has]: its row, and whether there is one."""
    i = torch.arange(max(n for n, _ in s["lens"]), device=_device())
    starts = s["q_start"].long()
    real = i < (starts[1:] - starts[:-1]).view(-1, 1)
    return torch.where(real, starts[:-1].view(-1, 1) + i, 0), real


def _plain_attend(s):
    c = s["case"]
    G, D, group, B = c["kv_heads"], c["dim"], c["heads"] // c["kv_heads"], c["seqs"]
    rows, real = _rows(s)
    N, length = rows.shape[1], max(n for _, n in s["lens"])
    at = s["kv_len"].long().view(-1, 1) - real.sum(1, keepdim=True) + torch.arange(N, device=_device())
    key = torch.arange(length, device=_device()).expand(B, -1)
    if c["window"] and c["sink"] + c["window"] + N < length:  # of a sequence what its rows see
        oldest = (at[:, :1] + 1 - c["window"]).clamp(min=c["sink"])
        key = torch.cat([key[:, :c["sink"]], oldest + torch.arange(c["window"] + N - 1, device=_device())], 1)
        length = key.shape[1]
    page = s["table"].gather(1, (key // c["page"]).clamp(max=s["table"].shape[1] - 1)).clamp(min=0).long()
    place = key % c["page"]
    k, v = ((_at(s[x])[page, :, place].view(CODES).float() *
             torch.exp2(_at(s[x + "_scale"])[page, :, place // BLOCK].float() - 127.0).unsqueeze(-1)) for x in "kv")
    q = s["q"][rows].float().view(B, N, G, group, D).permute(0, 2, 3, 1, 4).reshape(B * G, group * N, D)
    score = torch.bmm(q, k.permute(0, 2, 3, 1).reshape(B * G, D, length)).mul_(s["scale"]).view(B, G * group, N, length)
    key, at = key.view(B, 1, 1, length), at.view(B, 1, N, 1)
    hidden = key > at
    if c["window"]:
        hidden |= (key <= at - c["window"]) & (key >= c["sink"])
    score.masked_fill_(hidden, float("-inf"))
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.view(B * G, group * N, length), v.permute(0, 2, 1, 3).reshape(B * G, length, D))
    o = (o.view(B, G * group, N, D) / total).permute(0, 2, 1, 3).to(s["q"].dtype)
    out = torch.zeros_like(s["q"])
    out[rows[real]] = o[real]
    return {"out": out}


def _rotate(x, cos, sin, rot, inter):
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    y = x.clone()
    u, w = a * cos - b * sin, a * sin + b * cos
    if inter:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, w
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, w
    return y


def _store(s, name, x, seq, slots):
    """Rows x [row][head][dim] as codes: the scale of a block holds its new rows and, where it has some, is no less than
    it was for the rows that lie before them, whose codes follow it."""
    c = s["case"]
    codes, scales = _at(s[name]), _at(s[name + "_scale"])
    G, per = c["kv_heads"], c["page"] // BLOCK
    page = s["table"][seq, slots // c["page"]].long()
    block = page * per + slots % c["page"] // BLOCK
    top = torch.zeros(s[name].shape[0] * per, G, device=_device())
    top.scatter_reduce_(0, block.view(-1, 1).expand(-1, G), x.abs().amax(-1), "amax")
    # sequences whose first new row lies inside a block
    first = s["kv_len"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long()
    fpage = s["table"].gather(1, (first // c["page"]).view(-1, 1))[:, 0].long()
    start = first % c["page"] // BLOCK * BLOCK
    before = first % BLOCK
    was = scales[fpage, :, start // BLOCK].to(torch.int32) - 127
    e = _exponent(top).view(-1, per, G).transpose(1, 2).contiguous()  # [page][head][block]
    now = torch.where((before > 0).view(-1, 1), torch.maximum(was, e[fpage, :, start // BLOCK]), e[fpage, :, start // BLOCK])
    e[fpage, :, start // BLOCK] = now
    scales[page, :, slots % c["page"] // BLOCK] = (e[page, :, slots % c["page"] // BLOCK] + 127).to(torch.uint8)
    i = torch.arange(BLOCK, device=_device())
    old = (i < before.view(-1, 1)).nonzero()
    opage, oplace, grown = fpage[old[:, 0]], start[old[:, 0]] + old[:, 1], (was - now)[old[:, 0]]
    codes[opage, :, oplace] = _at(torch.ldexp(codes[opage, :, oplace].view(CODES).float(), grown.unsqueeze(-1)).to(CODES))
    codes[page, :, slots % c["page"]] = _at(torch.ldexp(x, -e[page, :, slots % c["page"] // BLOCK].unsqueeze(-1)).to(CODES))


def _plain_append(s):
    c = s["case"]
    H, G = c["heads"], c["kv_heads"]
    x = s["qkv"].float()
    count = (s["q_start"][1:] - s["q_start"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=_device()), count, output_size=x.shape[0])
    slots = torch.arange(x.shape[0], device=_device()) + (s["kv_len"].long() - s["q_start"][1:].long())[seq]
    angle = (slots if s["positions"] is None else s["positions"]).double().view(-1, 1, 1) * s["freqs"]
    cos, sin = (f.float() * s["mscale"] for f in (angle.cos(), angle.sin()))
    made = []
    for part, gain in ((x[:, :H], s["norm"][0]), (x[:, H:H + G], s["norm"][1])):
        if gain is not None:
            part = part * (part.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain
        made.append(_rotate(part, cos, sin, c["rot"], c["inter"]))
    _store(s, "k", made[1], seq, slots)
    _store(s, "v", x[:, H + G:], seq, slots)
    return {"q": made[0].to(s["qkv"].dtype), **{n: s[n] for n in ("k", "v", "k_scale", "v_scale")}}


def _plain_sample(s):
    c = s["case"]
    x, order = torch.sort(s["x"], dim=-1, descending=True, stable=True)
    t, top_p, min_p = (s["settings"][:, i:i + 1].double() for i in range(3))
    rank = torch.arange(c["vocab"], device=_device())
    w = ((x.double() - x[:, :1].double()) / torch.where(t > 0, t, 1.0)).exp()
    few = torch.where(t > 0, s["top_k"].view(-1, 1).long() if c["top_k"] else c["vocab"], 1)
    kept = rank < few
    run_sum = (w * kept).cumsum(-1)
    # of the top-p those before which the sum has not been reached
    kept &= (run_sum - w * kept < top_p * run_sum[:, -1:]) | (top_p >= 1.0)
    kept &= w >= min_p
    kept[:, 0] = True
    w = w * kept
    run_sum = w.cumsum(-1)
    total = run_sum[:, -1:]
    n = (run_sum <= s["uniform"].double().view(-1, 1) * total).sum(-1, keepdim=True).clamp(max=c["vocab"] - 1)
    return {"choice": order.gather(1, n)[:, 0].to(torch.int32), "prob": (w.gather(1, n) / total)[:, 0].float()}


PLAIN = {"attend": _plain_attend, "append": _plain_append, "sample": _plain_sample}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return PLAIN[kind](s)
    _run_own(s)
    if kind == "attend":
        return {"out": s["out"]}
    if kind == "append":
        return {"q": s["out"], "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return {"choice": s["choice"], "prob": s["prob"]}


# ---------------------------------------------------------------- 64 bits --
def _exact_attend(c, s):
    """Softmax by the logarithm of its sum, one head and a few hundred rows at a time."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_device())
    for b, (n, length) in enumerate(s["lens"]):
        where = torch.arange(length, device=_device())
        page, place = s["table"][b][where // c["page"]].long(), where % c["page"]
        for h in range(c["heads"]):
            g = h * c["kv_heads"] // c["heads"]
            k, v = (_at(s[x])[page, g, place].view(CODES).double() *
                    torch.pow(2.0, _at(s[x + "_scale"])[page, g, torch.div(place, 16, rounding_mode="floor")].double() - 127).view(-1, 1)
                    for x in "kv")
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                z = torch.mm(s["q"][s["starts"][b] + lo:s["starts"][b] + hi, h].double(), k.t()) * s["scale"]
                last = length - n + torch.arange(lo, hi, device=_device()).view(-1, 1)
                seen = where <= last
                if c["window"]:
                    seen &= (where > last - c["window"]) | (where < c["sink"])
                z = torch.where(seen, z, -math.inf)
                out[s["starts"][b] + lo:s["starts"][b] + hi, h] = torch.mm(torch.exp(z - torch.logsumexp(z, 1, keepdim=True)), v)
    return {"out": out}


def _e4m3(x):
    """To the nearest e4m3 number, ties to the even one: steps of 2^-3 of the value's power of two, of 2^-9 below 2^-6."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(c, s):
    """The pairs as complex numbers, turned; the pages' blocks one after the other."""
    H, G, rot = c["heads"], c["kv_heads"], c["rot"]
    x = s["qkv"].double()
    slot = torch.cat([torch.arange(length - n, length, device=_device()) for n, length in s["lens"]])
    pos = (slot if s["positions"] is None else s["positions"]).double()
    f = torch.tensor(frequencies(c)[0], dtype=torch.float64, device=_device())
    turn = torch.polar(torch.full((len(slot), rot // 2), float(s["mscale"]), dtype=torch.float64, device=_device()), torch.outer(pos, f))
    order = torch.arange(rot, device=_device())
    order = order.view(-1, 2) if c["inter"] else order.view(2, -1).t()
    for lo, hi, gain in ((0, H, s["norm"][0]), (H, H + G, s["norm"][1])):
        y = x[:, lo:hi]
        if gain is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / c["dim"] + EPS) * gain.double()
        z = torch.complex(y[..., order[:, 0]], y[..., order[:, 1]]) * turn.unsqueeze(1)
        y = y.clone()
        y[..., order[:, 0]], y[..., order[:, 1]] = z.real, z.imag
        x[:, lo:hi] = y
    out = {"q": x[:, :H].contiguous()}
    for name, new in (("k", x[:, H:H + G]), ("v", x[:, H + G:])):
        codes, scale = s[name].double(), torch.pow(2.0, _at(s[name + "_scale"]).double() - 127)
        for b, (n, length) in enumerate(s["lens"]):
            for block in range((length - n) // 16, (length - 1) // 16 + 1):
                lo, hi = max(16 * block, length - n), min(16 * block + 16, length)
                rows = new[s["starts"][b] + lo - (length - n):s["starts"][b] + hi - (length - n)]
                page, place = int(s["table"][b, 16 * block // c["page"]]), 16 * block % c["page"]
                need = torch.exp2(torch.ceil(torch.log2(rows.abs().amax((0, 2)) / 448.0)).clamp(min=-100))
                if lo > 16 * block:
                    was = scale[page, :, place // 16].clone()
                    need = torch.maximum(need, was)
                    old = slice(place, place + lo - 16 * block)
                    codes[page, :, old] = _e4m3(codes[page, :, old] * (was / need).view(-1, 1, 1))
                scale[page, :, place // 16] = need
                codes[page, :, place + lo - 16 * block:place + hi - 16 * block] = _e4m3((rows / need.view(1, -1, 1)).transpose(0, 1))
        out[name], out[name + "_scale"] = codes, scale
    return out


def _exact_sample(c, s):
    """Row by row, with numbers of the row's own kept set only."""
    prob = []
    for r in range(c["rows"]):
        t, top_p, min_p = (float(a) for a in s["settings"][r])
        x = s["x"][r].double()
        if t <= 0:
            prob.append(1.0)
            continue
        order = torch.argsort(-x, stable=True)[:int(s["top_k"][r]) if c["top_k"] else c["vocab"]]
        share = torch.softmax(x[order] / t, 0)
        before = torch.cat([share.new_zeros(1), share.cumsum(0)[:-1]])
        n = len(order) if top_p >= 1 else max(1, int((before < top_p * share.sum()).sum()))
        n = max(1, min(n, int((share >= min_p * share[0]).sum())))
        share = share[:n] / share[:n].sum()
        at = int(torch.searchsorted(share.cumsum(0), float(s["uniform"][r]), right=True))
        prob.append(float(share[min(at, n - 1)]))
    return {"choice": None, "prob": torch.tensor(prob, dtype=torch.float64, device=_device())}


def exact(case, seed):
    s = PREPARE[case["kind"]](case, _Draws(seed))
    return {"attend": _exact_attend, "append": _exact_append, "sample": _exact_sample}[case["kind"]](case, s)
