"""The operators a serving program puts between its projections and its next token, as measurable cases.

A program that decodes several recordings at once keeps their keys and values in pages of one
pool and runs, for each step, the new rows of all of them together:

  rope     mtg_rope_append_dev: the rows of the fused q|k|v product get their rotary positions
           (after the decoder's q / k norms where it has them); q goes on, k and v go into the pages
  attend   mtg_paged_attn_dev: causal attention of the new rows over the pages
  logits   mtg_logits_step_dev: penalties for repeated tokens, biases and grammar masks on the
           rows of logits, and the first-max choice of what remains

Sizes are this library's own decoder (16 / 8 heads of 128, 151,936 ids), its contexts (512 to
16,384 positions) and verify widths, and other head layouts of the same range. Sequences of a
batch have different lengths. Types are the library's: rows in f32 or f16, caches in f32 or f16.

With `own` false, run() computes the operators from elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f32": torch.float32, "f16": torch.float16}
BYTES = {"f32": 4, "f16": 2}
EPS = 1e-6
ROPE_BASE = 1e6
GOLDEN = 0.6180339887498949


def listed():
    return [
        # one recording, one token at a time: the smallest step there is
        dict(name="attend_1x1_613", kind="attend", io="f32", kv="f16", heads=16, kv_heads=8, dim=128, page=16,
             seqs=1, new=1, ctx=613, window=0),
        # a batch of recordings of all ages, one token each
        dict(name="attend_24x1_8000", kind="attend", io="f16", kv="f16", heads=16, kv_heads=8, dim=128, page=16,
             seqs=24, new=1, ctx=8000, window=0),
        # seven drafts and their seed for each of eight recordings, f32 cache
        dict(name="attend_8x8_4000_f32", kind="attend", io="f32", kv="f32", heads=16, kv_heads=8, dim=128, page=32,
             seqs=8, new=8, ctx=4000, window=0),
        # a block of a long prompt with the library's own types (f32 rows, f16 cache), ragged
        dict(name="attend_1x1009_7963", kind="attend", io="f32", kv="f16", heads=16, kv_heads=8, dim=128, page=64,
             seqs=1, new=1009, ctx=7963, window=0),
        # blocks of two long prompts, f16 throughout, a wide model's heads
        dict(name="attend_2x2048_16384", kind="attend", io="f16", kv="f16", heads=32, kv_heads=8, dim=128, page=64,
             seqs=2, new=2048, ctx=16384, window=0),
        # one new row of the library's decoder: norms, whole-head half pairs, f16 cache
        dict(name="rope_1x1", kind="rope", io="f32", kv="f16", heads=16, kv_heads=8, dim=128, page=16, seqs=1, new=1,
             ctx=613, rot=128, inter=False, factor=1.0, norm=True),
        # interleaved pairs on half of the head, a context stretched eight times, far positions, f32 cache
        dict(name="rope_48x13_far", kind="rope", io="f32", kv="f32", heads=24, kv_heads=4, dim=128, page=32, seqs=48,
             new=13, ctx=2000, rot=64, inter=True, factor=8.0, norm=False),
        # the rows of a whole long prompt, f16 throughout
        dict(name="rope_1x16384", kind="rope", io="f16", kv="f16", heads=16, kv_heads=8, dim=128, page=64, seqs=1,
             new=16384, ctx=0, rot=128, inter=False, factor=1.0, norm=True),
        # the one row of a sampled step: penalties over the last hundred ids, the row goes to the sampler
        dict(name="logits_1", kind="logits", io="f32", rows=1, vocab=151936, hist=100, bias=8, mask=False, out=True),
        # sixteen verify rows, only the choices are wanted
        dict(name="logits_16_choice", kind="logits", io="f32", rows=16, vocab=151936, hist=100, bias=0, mask=False,
             out=False),
        # a batch under a grammar, long histories, f16, an odd vocabulary
        dict(name="logits_61_grammar_f16", kind="logits", io="f16", rows=61, vocab=151643, hist=2000, bias=64, mask=True,
             out=True),
        # a large batch with everything
        dict(name="logits_256_grammar", kind="logits", io="f32", rows=256, vocab=151936, hist=1000, bias=300, mask=True,
             out=True),
    ]


def draw(rng):
    """A case of the same ranges. What costs more than the largest listed case of its kind is drawn again."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = {k: [max(work(c)[w] for c in listed() if c["kind"] == k) for w in ("bytes", "flops")]
            for k in ("attend", "rope", "logits")}
    while True:
        kind = rng.choice(["attend", "attend", "rope", "logits"])
        if kind == "logits":
            case = dict(kind=kind, io=rng.choice(["f32", "f16"]), rows=log_int(1, 256), vocab=log_int(1000, 151936),
                        hist=log_int(1, 4000), bias=rng.choice([0, log_int(1, 300)]), mask=rng.random() < 0.5,
                        out=rng.random() < 0.75)
        else:
            io, kv = rng.choice([("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
            kv_heads = rng.choice([1, 2, 4, 8])
            case = dict(kind=kind, io=io, kv=kv, heads=kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv_heads,
                        dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128, 256]), seqs=log_int(1, 64),
                        new=rng.choice([1, log_int(2, 16), log_int(17, 2048)]), ctx=log_int(1, 32768))
            if kind == "attend":
                case["window"] = rng.choice([0, 0, 0, log_int(16, 8192)])
            else:
                case.update(rot=rng.choice([case["dim"], case["dim"] // 2, 2 * log_int(4, case["dim"] // 2)]),
                            inter=rng.random() < 0.5, factor=rng.choice([1.0, 4.0, 16.0]), norm=rng.random() < 0.5)
        w = work(case)
        if w["bytes"] <= most[kind][0] and w["flops"] <= max(most[kind][1], 1) and pool_bytes(case) < 3 << 30:
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
    if case["kind"] == "logits":
        return 0
    return 2 * (sum(pages_of(case)) + 3) * case["page"] * case["kv_heads"] * case["dim"] * BYTES[case["kv"]]


def work(case):
    """Each input read once, each output written once."""
    if case["kind"] == "logits":
        b = BYTES[case["io"]]
        row = case["vocab"] * b * (2 if case["out"] else 1) + 4 * case["hist"] + 8 * case["bias"] + 4
        row += -(-case["vocab"] // 32) * 4 if case["mask"] else 0
        return {"bytes": case["rows"] * row, "flops": 3 * case["rows"] * case["vocab"]}
    io, kv, d = BYTES[case["io"]], BYTES[case["kv"]], case["dim"]
    rows = sum(n for n, _ in lengths(case))
    if case["kind"] == "rope":
        moved = rows * d * (io * (2 * case["heads"] + 2 * case["kv_heads"]) + kv * 2 * case["kv_heads"])
        return {"bytes": moved, "flops": rows * (case["heads"] + case["kv_heads"]) * (3 * case["rot"] + 4 * d * case["norm"])}
    read, seen = 0, 0
    for n, length in lengths(case):
        w = case["window"] if case["window"] else length
        first = max(0, length - n + 1 - w)  # the first row's oldest key
        read += length - first
        seen += sum(min(length - n + 1 + i, w) for i in range(n))
    return {"bytes": 2 * read * case["kv_heads"] * d * kv + 2 * rows * case["heads"] * d * io,
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

    def ints(self, hi, *shape):
        return torch.randint(0, hi, shape, generator=self.g, device=_device(), dtype=torch.int32)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=_device(), dtype=torch.int64).to(torch.int32)


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


def _cache(case, r):
    """Pages of a pool in no order, the sequences' tables (no row of them is full), and their lengths."""
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
    shape = (pool, case["kv_heads"], case["page"], case["dim"])
    dtype = DTYPES[case["kv"]]
    return dict(lens=lens, starts=starts, table=table, q_start=_ints(starts), kv_len=_ints([length for _, length in lens]),
                k=r.normal(*shape, dtype=dtype), v=r.normal(*shape, dtype=dtype))


def _prepare_attend(case, r):
    s = _cache(case, r)
    # rows as a rotated, normed q has them: unit variance, some heads sharper than others
    sharp = torch.linspace(0.5, 2.5, case["heads"], device=_device()).view(1, -1, 1)
    s["q"] = (r.normal(s["starts"][-1], case["heads"], case["dim"]) * sharp).to(DTYPES[case["io"]])
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    return s


def _prepare_rope(case, r):
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


def _prepare_logits(case, r):
    rows, vocab = case["rows"], case["vocab"]
    s = {"x": (3.0 * r.normal(rows, vocab)).to(DTYPES[case["io"]])}
    # the histories of the rows one after the other; a quarter of the ids come again and again
    h = r.ints(vocab, rows * case["hist"])
    often = r.ints(max(1, min(vocab, 40)), rows * case["hist"])
    s["history"] = torch.where(r.ints(4, rows * case["hist"]) == 0, often, h)
    at = torch.arange(rows, dtype=torch.int32, device=_device())
    s["hist_range"] = torch.stack([at * case["hist"], (at + 1) * case["hist"]], 1).contiguous()
    s["penalties"] = torch.tensor([[1.1, 0.1, 0.2]], device=_device()).repeat(rows, 1) + 0.05 * r.ints(4, rows, 3)
    if case["bias"]:  # the requests' own lists: no id twice in a list
        n = min(case["bias"], vocab)
        s["bias_ids"] = torch.cat([r.order(vocab)[:n] for _ in range(rows)])
        s["bias"] = 2.0 * r.normal(rows * n)
        s["bias_range"] = torch.stack([at * n, (at + 1) * n], 1).contiguous()
    if case["mask"]:  # bit i of word w: id 32 w + i may follow
        s["mask"] = r.ints(1 << 30, rows, -(-vocab // 32)) | (r.ints(4, rows, -(-vocab // 32)) << 30)
    return s


def prepare(case, seed):
    r = _Draws(seed)
    s = {"attend": _prepare_attend, "rope": _prepare_rope, "logits": _prepare_logits}[case["kind"]](case, r)
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
    if case["kind"] == "logits":
        s["out"] = torch.empty_like(s["x"]) if case["out"] else None
        s["choice"] = torch.empty(case["rows"], dtype=torch.int32, device=_device())
        d = mtg.LogitsStep(logits=at(s["x"]), out=at(s["out"]), stride=case["vocab"], out_stride=case["vocab"],
                           history=at(s["history"]), hist_range=at(s["hist_range"]), penalties=at(s["penalties"]),
                           choice=at(s["choice"]), io_type=types[case["io"]], rows=case["rows"], vocab=case["vocab"],
                           n_history=s["history"].numel())
        if case["bias"]:
            d.bias_ids, d.bias, d.bias_range, d.n_bias = at(s["bias_ids"]), at(s["bias"]), at(s["bias_range"]), s["bias"].numel()
        if case["mask"]:
            d.mask, d.mask_stride = at(s["mask"]), s["mask"].shape[1]
        s["call"], size = L.mtg_logits_step_dev, L.mtg_logits_step_workspace(ctypes.byref(d))
    else:
        H, D, width = case["heads"], case["dim"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        kv = mtg.PagedKv(k=at(s["k"]), v=at(s["v"]), page_table=at(s["table"]), kv_len=at(s["kv_len"]),
                         q_start=at(s["q_start"]), page_stride=case["kv_heads"] * case["page"] * D,
                         head_stride=case["page"] * D, kv_type=types[case["kv"]], n_pages=s["k"].shape[0],
                         page_size=case["page"], table_stride=s["table"].shape[1], n_seqs=case["seqs"],
                         n_tokens=s["starts"][-1], n_kv_heads=case["kv_heads"], head_dim=D)
        if case["kind"] == "attend":
            s["out"] = torch.empty_like(s["q"])
            d = mtg.PagedAttn(kv=kv, q=at(s["q"]), out=at(s["out"]), q_stride=H * D, out_stride=H * D,
                              io_type=types[case["io"]], n_heads=H, max_kv=max(length for _, length in s["lens"]),
                              window=case["window"], scale=s["scale"])
            s["call"], size = L.mtg_paged_attn_dev, L.mtg_paged_attn_workspace(ctypes.byref(d))
        else:
            s["out"] = torch.empty(s["starts"][-1], H, D, dtype=s["qkv"].dtype, device=_device())
            x, b = at(s["qkv"]), BYTES[case["io"]]
            d = mtg.RopeAppend(kv=kv, q=x, k_new=x + H * D * b, v_new=x + (H + case["kv_heads"]) * D * b,
                               q_out=at(s["out"]), positions=at(s["positions"]), freqs=at(s["freqs"]),
                               q_norm=at(s["norm"][0]), k_norm=at(s["norm"][1]), q_stride=width, k_stride=width,
                               v_stride=width, q_out_stride=H * D, io_type=types[case["io"]], n_heads=H,
                               rot_dim=case["rot"], interleaved=int(case["inter"]), eps=EPS, mscale=s["mscale"])
            s["call"], size = L.mtg_rope_append_dev, 0
    if size:
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device=_device())
        d.workspace, d.workspace_bytes = at(s["workspace"]), size
    s["desc"], s["arg"] = d, ctypes.byref(d)


def _run_own(s):
    rc = s["call"](s["arg"], s["stream"])
    if rc:
        raise RuntimeError("status %d" % rc)


# ------------------------------------------------------------- plain forms --
def _slots(s, b):
    n, length = s["lens"][b]
    return torch.arange(length - n, length, device=_device())


def _plain_attend(s):
    c = s["case"]
    group, out = c["heads"] // c["kv_heads"], torch.zeros_like(s["q"])
    for b, (n, length) in enumerate(s["lens"]):
        ids = s["table"][b, :-(-length // c["page"])].long()
        k, v = (s[x][ids].transpose(0, 1).reshape(c["kv_heads"], -1, c["dim"])[:, :length].float() for x in "kv")
        rows = slice(s["starts"][b], s["starts"][b + 1])
        q = s["q"][rows].float().view(n, c["kv_heads"], group, c["dim"]).permute(1, 2, 0, 3)
        score = (q.reshape(c["kv_heads"], group * n, c["dim"]) @ k.transpose(1, 2)).mul_(s["scale"])
        score = score.view(c["kv_heads"], group, n, length)
        key, at = torch.arange(length, device=_device()), _slots(s, b).view(-1, 1)
        hidden = (key > at) if not c["window"] else (key > at) | (key <= at - c["window"])
        score.masked_fill_(hidden, float("-inf"))
        p = (score - score.amax(-1, keepdim=True)).exp_()
        o = (p.view(c["kv_heads"], group * n, length) @ v).view(c["kv_heads"], group, n, c["dim"]) / p.sum(-1, keepdim=True)
        out[rows] = o.permute(2, 0, 1, 3).reshape(n, c["heads"], c["dim"]).to(out.dtype)
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


def _plain_rope(s):
    c = s["case"]
    H, G = c["heads"], c["kv_heads"]
    x = s["qkv"].float()
    slots = torch.cat([_slots(s, b) for b in range(c["seqs"])])
    at = slots if s["positions"] is None else s["positions"]
    angle = at.double().view(-1, 1, 1) * s["freqs"]
    cos, sin = (f.float() * s["mscale"] for f in (angle.cos(), angle.sin()))
    made = []
    for part, gain in ((x[:, :H], s["norm"][0]), (x[:, H:H + G], s["norm"][1])):
        if gain is not None:
            part = part * (part.square().mean(-1, keepdim=True) + EPS).rsqrt() * gain
        made.append(_rotate(part, cos, sin, c["rot"], c["inter"]))
    seq = torch.repeat_interleave(torch.arange(c["seqs"], device=_device()),
                                  torch.tensor([n for n, _ in s["lens"]], device=_device()))
    page = s["table"][seq, slots // c["page"]].long()
    s["k"][page, :, slots % c["page"]] = made[1].to(s["k"].dtype)
    s["v"][page, :, slots % c["page"]] = x[:, H + G:].to(s["v"].dtype)
    return {"q": made[0].to(s["qkv"].dtype), "k": s["k"], "v": s["v"]}


def _plain_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    y = s["x"].float()
    row = torch.arange(rows, device=_device()).view(-1, 1)
    count = torch.zeros(rows, vocab, device=_device())
    count.view(-1).index_add_(0, (row * vocab + s["history"].view(rows, -1)).view(-1), torch.ones(s["history"].numel(), device=_device()))
    rep, freq, pres = (s["penalties"][:, i:i + 1] for i in range(3))
    y = torch.where(count > 0, torch.where(y > 0, y / rep, y * rep) - (freq * count + pres), y)
    if c["bias"]:
        y[row, s["bias_ids"].view(rows, -1).long()] += s["bias"].view(rows, -1)
    if c["mask"]:
        bits = (s["mask"].unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=_device())) & 1
        y = torch.where(bits.view(rows, -1)[:, :vocab] == 1, y, float("-inf"))
    y = y.to(s["x"].dtype)
    best = y == y.amax(-1, keepdim=True)
    index = torch.arange(vocab, dtype=torch.int32, device=_device())
    choice = torch.where(best, index, vocab).amin(-1).to(torch.int32)
    return {"out": y if c["out"] else None, "choice": choice}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"attend": _plain_attend, "rope": _plain_rope, "logits": _plain_logits}[kind](s)
    _run_own(s)
    if kind == "attend":
        return {"out": s["out"]}
    if kind == "rope":
        return {"q": s["out"], "k": s["k"], "v": s["v"]}
    return {"out": s["out"], "choice": s["choice"]}


# ---------------------------------------------------------------- 64 bits --
def _exact_attend(c, s):
    """Softmax by the logarithm of its sum, one head and a few hundred rows at a time."""
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=_device())
    for b, (n, length) in enumerate(s["lens"]):
        where = torch.arange(length, device=_device())
        page, place = s["table"][b][where // c["page"]].long(), where % c["page"]
        for h in range(c["heads"]):
            g = h * c["kv_heads"] // c["heads"]
            k, v = s["k"][page, g, place].double(), s["v"][page, g, place].double()
            for lo in range(0, n, 512):
                hi = min(n, lo + 512)
                z = torch.mm(s["q"][s["starts"][b] + lo:s["starts"][b] + hi, h].double(), k.t()) * s["scale"]
                last = length - n + torch.arange(lo, hi, device=_device()).view(-1, 1)
                seen = where <= last
                if c["window"]:
                    seen &= where > last - c["window"]
                z = torch.where(seen, z, -math.inf)
                out[s["starts"][b] + lo:s["starts"][b] + hi, h] = torch.mm(torch.exp(z - torch.logsumexp(z, 1, keepdim=True)), v)
    return {"out": out}


def _exact_rope(c, s):
    """The pairs as complex numbers, turned; row by row places in the pool."""
    H, G, rot = c["heads"], c["kv_heads"], c["rot"]
    x = s["qkv"].double()
    place = [(b, length - n + i) for b, (n, length) in enumerate(s["lens"]) for i in range(n)]
    slot = torch.tensor([p for _, p in place], device=_device())
    page = s["table"][torch.tensor([b for b, _ in place], device=_device()), torch.div(slot, c["page"], rounding_mode="floor")].long()
    pos = (slot if s["positions"] is None else s["positions"]).double()
    f = torch.tensor(frequencies(c)[0], dtype=torch.float64, device=_device())
    turn = torch.polar(torch.full((len(place), rot // 2), float(s["mscale"]), dtype=torch.float64, device=_device()), torch.outer(pos, f))
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
    k, v = s["k"].double(), s["v"].double()
    k[page, :, slot % c["page"]] = x[:, H:H + G]
    v[page, :, slot % c["page"]] = x[:, H + G:]
    return {"q": x[:, :H].contiguous(), "k": k, "v": v}


def _exact_logits(c, s):
    """Row by row, only the ids that a list names."""
    if not c["out"]:  # an index is not a computed number: the plain form's has to be met
        return None
    y = s["x"].double()
    for r in range(c["rows"]):
        ids, times = torch.unique(s["history"][r * c["hist"]:(r + 1) * c["hist"]].long(), return_counts=True)
        rep, freq, pres = s["penalties"][r].double()
        z = y[r, ids]
        y[r, ids] = torch.where(z > 0, z / rep, z * rep) - freq * times - pres
        if c["bias"]:
            lo, hi = (int(i) for i in s["bias_range"][r])
            y[r].index_add_(0, s["bias_ids"][lo:hi].long(), s["bias"][lo:hi].double())
        if c["mask"]:
            ids = torch.arange(c["vocab"], device=_device())
            y[r, ((s["mask"][r, ids // 32] >> (ids % 32).to(torch.int32)) & 1) == 0] = -math.inf
    return {"out": y, "choice": None}


def exact(case, seed):
    r = _Draws(seed)
    s = {"attend": _prepare_attend, "rope": _prepare_rope, "logits": _prepare_logits}[case["kind"]](case, r)
    return {"attend": _exact_attend, "rope": _exact_rope, "logits": _exact_logits}[case["kind"]](case, s)
