"""Measured cases of four operators of a decoding step: queries and keys normalised for each head and turned by their
positions in one pass, the 4-bit paged key/value cache as it is written and read back, the attention over it, and the
products of a few rows with 4-bit weights.

listed() and draw() give the cases, prepare() a program's data on the GPU, run() one pass through an operator: in its
plain form (elementary torch operations) where `own` is false, by the library's calls where it is true.  exact() is the
operators' definition in 64 bits.

The backend launches on a stream of its own, which waits for no other.  A program that makes its inputs with torch
makes that stream torch's current one, as prepare() does, and everything is in order; where another stream is current
when run() is called, the two wait for each other around the calls.  Results are ready on the current stream.

The cache: 32 consecutive dimensions of one token's head share a scale, the element of largest magnitude (the positive
one of two) divided by -8 and rounded to bf16; a code is the quotient rounded to nearest even and cut to -8 .. 7, held as
code + 8 in 4 bits, dimension 2 i in the low half of byte i.  Codes uint8 [pages][kv heads][page tokens][head dim / 2],
scales bf16 [pages][kv heads][page tokens][head dim / 32].  A sequence's tokens [i P, (i + 1) P) lie in the page that entry
i of its row of the block table names.  A batch gives each sequence a run of rows (row_start) and its length with these
rows (kv_len): its rows are its last tokens.

The weights: ggml's blocks of 32 along a row, Q4_0 {f16 d, 16 bytes} with the value d (code - 8) and Q4_1 {f16 d, f16 m,
16 bytes} with the value d code + m; byte j holds element j in its low half and element j + 16 in its high one.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
SMALL = 2.0 ** -100  # groups of the cache whose largest value is below this hold zeros

_kept = {}


def _framework():
    """The package's bindings and one backend on the GPU, as a program keeps them."""
    if "be" not in _kept:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location("sam3_b200_b200", os.path.join(root, "sam3.cpp_b200", "b200.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[spec.name] = mod
        spec.loader.exec_module(mod)
        _kept["mod"], _kept["be"] = mod, mod.Backend(torch.cuda.current_device())
        _kept["attend"] = _kept["be"].kv_attention()
        _kept["stream"] = torch.cuda.ExternalStream(_kept["be"].stream)
    return _kept["mod"], _kept["be"]


# ---- cases -----------------------------------------------------------------------------------------------------


def listed():
    norm = dict(op="norm", kind="rms", sections="64", pairing="halves", deal=False, restart=False, base=1e6, first=0, text=0,
                frames=0, height=0, width=0, type="bf16", out="bf16")
    cache = dict(op="cache", kv_heads=8, dim=128, page=64, type="bf16")
    attend = dict(op="attend", heads=32, kv_heads=8, dim=128, page=64, type="bf16", causal=True, window=0)
    vec = dict(op="vec", weights="q4_0", bias=False)
    return [
        # one token of each of 9 sequences: queries and keys of the layer's projection
        dict(norm, name="norm_step", text=9, q_heads=32, k_heads=8, dim=128, first=20000),
        # the 72 x 72 tokens of one image: layer norms, two axes with frequencies of their own, f32 -> f16
        dict(norm, name="norm_image", kind="layer", frames=1, height=72, width=72, q_heads=16, k_heads=16, dim=64,
             sections="0,16,16", pairing="neighbours", restart=True, base=1e4, type="f32", out="f16"),
        # a video prompt of 9 frames between text
        dict(norm, name="norm_video", text=301, frames=9, height=36, width=64, q_heads=32, k_heads=8, dim=128,
             sections="24,20,20", deal=True, first=1000),
        # every sequence of a serving batch appends one token, its last page is read back
        dict(cache, name="cache_step", seqs=80, new=1, new_max=1, past=100, past_max=4000, read="page"),
        # ragged prompts appended behind earlier ones, the whole contexts read back
        dict(cache, name="cache_prompt", seqs=6, new=800, new_max=4200, past=0, past_max=1700, page=16, type="f16", read="all"),
        # a single token of a single short sequence: latency
        dict(attend, name="attend_one", seqs=1, new=1, new_max=1, past=900, past_max=900),
        # a serving batch, one token each, ragged lengths
        dict(attend, name="attend_batch", seqs=64, new=1, new_max=1, past=1000, past_max=16100),
        # several drafted tokens of each of a few long contexts, heads without groups
        dict(attend, name="attend_few", seqs=4, new=3, new_max=5, past=30000, past_max=70000, heads=8, kv_heads=8, dim=64, page=128,
             type="f16"),
        # parts of prompts behind earlier contexts
        dict(attend, name="attend_chunk", seqs=4, new=300, new_max=900, past=2000, past_max=7000, kv_heads=4, page=32, type="f16"),
        # a text encoder's MLP for one token, activations f32 as the graph's nodes have them
        dict(vec, name="vec_small", rows=1, k=1024, n=4096, bias=True, type="f32", out="f32"),
        # a wide layer of a step of 6 sequences
        dict(vec, name="vec_rows", weights="q4_1", rows=6, k=4096, n=14339, type="bf16", out="bf16"),
        # the logits of one token over the text encoder's vocabulary
        dict(vec, name="vec_logits", rows=1, k=4096, n=49408, type="f16", out="f32"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "cache", "attend", "attend", "vec", "vec"])
    dim = rng.choice([64, 128, 128])
    if op == "norm":
        dim = rng.choice([64, 80, 128, 128, 256])
        pairs = dim // 2
        axes = rng.choice([1, 1, 2, 3, 4])
        cut = sorted(rng.randint(1, pairs - 1) for _ in range(axes - 1))
        sections = [b - a for a, b in zip([0] + cut, cut + [pairs])]
        if rng.random() < 0.2:  # a part of each head is not turned
            sections[-1] = (sections[-1] + 1) // 2
        k_heads = rng.choice([1, 2, 4, 8, 8])
        return dict(op="norm", kind=rng.choice(["rms", "rms", "layer"]), text=_log_int(rng, 1, 3000),
                    frames=rng.choice([0, 1, rng.randint(2, 6)]), height=rng.randint(5, 36), width=rng.randint(5, 48),
                    q_heads=k_heads * rng.randint(1, 4), k_heads=k_heads, dim=dim, sections=",".join(map(str, sections)),
                    pairing=rng.choice(["halves", "neighbours"]), deal=rng.random() < 0.5, restart=rng.random() < 0.3,
                    base=rng.choice([1e4, 5e5, 1e6]), first=rng.choice([0, _log_int(rng, 10, 500000)]),
                    type=rng.choice(["bf16", "f16", "f32"]), out=rng.choice(["bf16", "f16", "f32"]))
    if op == "vec":
        rows = rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(2, 16)])
        k = 32 * _log_int(rng, 2, 512)
        n = _log_int(rng, 5, min(60000, 100000000 // (k * (1 + rows // 5))))
        t = rng.choice(["bf16", "f16", "f32"])
        return dict(op="vec", weights=rng.choice(["q4_0", "q4_0", "q4_1"]), rows=rows, k=k, n=n, bias=rng.random() < 0.4, type=t,
                    out=rng.choice([t, "f32"]))
    page, kv_heads = rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8, 8, 16])
    if op == "cache":
        if rng.random() < 0.5:
            seqs, new, new_max, past_max = _log_int(rng, 1, 96), 1, rng.randint(1, 8), _log_int(rng, 10, 4000)
            read = "page"
        else:
            seqs = rng.randint(1, 6)
            new = _log_int(rng, 8, 2000)
            new_max, past_max, read = min(4000, 2 * new + 1), _log_int(rng, 1, 3000), rng.choice(["page", "all"])
            kv_heads = min(kv_heads, 8)
        return dict(op="cache", kv_heads=kv_heads, dim=dim, page=page, type=rng.choice(["bf16", "f16", "f32"]), seqs=seqs, new=new,
                    new_max=new_max, past=0, past_max=past_max, read=read)
    kind = rng.choice(["step", "step", "few", "prompt", "cross"])
    group = rng.choice([1, 2, 3, 4, 5, 8, 16])
    kv_heads = min(kv_heads, 48 // group)
    window = rng.choice([0, 0, _log_int(rng, 20, 3000)])
    if kind == "step":
        seqs = _log_int(rng, 1, 64)
        new = new_max = 1
        past_max = _log_int(rng, 60, min(100000, 500000 // seqs))
    elif kind == "few":
        seqs, new, new_max = _log_int(rng, 1, 24), 2, rng.randint(3, 9)
        past_max = _log_int(rng, 60, min(30000, 150000 // seqs))
    elif kind == "prompt":
        seqs = rng.randint(1, 4)
        new = _log_int(rng, 20, 2200 // seqs)
        new_max, past_max = min(2500, new + new // 2 + 1), _log_int(rng, 1, 2200)
    else:
        seqs, new = rng.randint(1, 2), _log_int(rng, 10, 2200)
        new_max, past_max, window = new + 7, _log_int(rng, 100, 2200), 0
    return dict(op="attend", heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page, type=rng.choice(["bf16", "f16"]),
                causal=kind != "cross", window=window, seqs=seqs, new=new, new_max=new_max, past=past_max // 2, past_max=past_max)


# ---- a program's data ------------------------------------------------------------------------------------------


def _lengths(case):
    """New rows and earlier tokens of each sequence: part of the case, the same for every seed."""
    r = random.Random("%s %s %s" % (case["seqs"], case["new_max"], case["past_max"]))
    new = [r.randint(case["new"], case["new_max"]) for _ in range(case["seqs"])]
    past = [r.randint(case["past"], case["past_max"]) for _ in range(case["seqs"])]
    return new, past


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _sections(case):
    return [int(x) for x in case["sections"].split(",")]


def _tokens(case):
    return case["text"] + case["frames"] * case["height"] * case["width"]


def _norm_data(case, g):
    """Half of the text, the frames' grid, the rest of the text.  The rows hold queries, keys and values side by side."""
    n, t = _tokens(case), TYPES[case["type"]]
    before = case["text"] // 2
    f, h, w = case["frames"], case["height"], case["width"]
    lead = torch.arange(before).expand(4, before)
    grid = torch.stack([x.reshape(-1) for x in torch.meshgrid(torch.arange(f), torch.arange(h), torch.arange(w), indexing="ij")])
    grid = torch.cat([grid, grid[:1]]) + before
    rest = torch.arange(case["text"] - before).expand(4, -1) + (before + max(f, h, w) if f else before)
    pos = torch.cat([lead, grid, rest], 1)[: len(_sections(case))] + case["first"]
    hq, hk, d = case["q_heads"], case["k_heads"], case["dim"]
    # heads differ in size, some channels stand out
    size = torch.exp(0.5 * torch.randn(hq + 2 * hk, 1, generator=g, device="cuda") + 0.5 * torch.randn(1, d, generator=g, device="cuda"))
    st = {"x": (torch.randn(n, hq + 2 * hk, d, generator=g, device="cuda") * size).to(t), "pos": pos.to(torch.int32).contiguous().cuda()}
    for name, heads in (("q", hq), ("k", hk)):
        st[name + "_weight"] = 1 + 0.2 * torch.randn(d, generator=g, device="cuda")
        st[name + "_bias"] = 0.1 * torch.randn(d, generator=g, device="cuda") if case["kind"] == "layer" else None
        st[name + "_out"] = torch.empty(n, heads, d, dtype=TYPES[case["out"]], device="cuda")
    st["eps"] = 1e-6
    return st


def _cache_data(case, g):
    new, past = _lengths(case)
    heads, d, p, t = case["kv_heads"], case["dim"], case["page"], TYPES[case["type"]]
    total = [a + b for a, b in zip(new, past)]
    used = [-(-n // p) for n in total]
    width, pages = max(used) + 1, sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(len(new), width, dtype=torch.int32)
    at = 0
    for s, n in enumerate(used):
        table[s, :n] = order[at:at + n]
        at += n
    st = {"new": new, "total": total, "table": table.cuda(),
          "row_start": torch.tensor(_starts(new), dtype=torch.int32, device="cuda"),
          "kv_len": torch.tensor(total, dtype=torch.int32, device="cuda")}
    for name in ("k", "v"):
        st[name + "_codes"] = torch.randint(0, 256, (pages, heads, p, d // 2), generator=g, device="cuda", dtype=torch.uint8)
        # scales of either sign, as the largest element's sign decides
        size = torch.exp(0.3 * torch.randn(pages, heads, p, d // 32, generator=g, device="cuda")) * (0.25 if name == "k" else 0.2)
        st[name + "_scale"] = (size * torch.sign(torch.randn(size.shape, generator=g, device="cuda"))).to(torch.bfloat16)
    if case["op"] == "cache":
        read = [n if case["read"] == "all" else n - (b // p) * p for n, b in zip(total, past)]
        st["read"] = read
        st["read_start"] = torch.tensor(_starts(read), dtype=torch.int32, device="cuda")
        for name in ("k", "v"):
            # channels of keys differ in size
            size = torch.exp(0.6 * torch.randn(heads, d, generator=g, device="cuda")) if name == "k" else 1.0
            st[name] = (torch.randn(sum(new), heads, d, generator=g, device="cuda") * size).to(t)
            st[name + "_out"] = torch.empty(sum(read), heads, d, dtype=t, device="cuda")
    else:
        # queries of the size that spreads the softmax over some tens of keys
        st["q"] = (torch.randn(sum(new), case["heads"], d, generator=g, device="cuda") * 1.2).to(t)
        st["out"] = torch.empty_like(st["q"])
        st["scale"] = 1.0 / math.sqrt(d)
    return st


def _vec_data(case, g):
    """Blocks of normal weights as ggml quantises them, and rows of activations of which some channels stand out."""
    n, k, m = case["n"], case["k"], case["rows"]
    w = torch.randn(n * (k // 32), 32, generator=g, device="cuda") / math.sqrt(k)
    low, high = w.amin(1, keepdim=True), w.amax(1, keepdim=True)
    if case["weights"] == "q4_0":
        d = torch.where(high >= -low, high, low) / -8
        code = ((w / d).round() + 8).clamp_(0, 15).to(torch.uint8)
        head = [d]
    else:
        d = (high - low) / 15
        code = ((w - low) / d).round_().clamp_(0, 15).to(torch.uint8)
        head = [d, low]
    blocks = torch.cat([h.half().view(torch.uint8) for h in head] + [code[:, :16] | code[:, 16:] << 4], 1)
    del w, code
    size = torch.exp(0.7 * torch.randn(k, generator=g, device="cuda"))
    return {"blocks": blocks.contiguous(), "x": (torch.randn(m, k, generator=g, device="cuda") * size).to(TYPES[case["type"]]),
            "bias": 0.1 * torch.randn(n, generator=g, device="cuda") if case["bias"] else None,
            "out": torch.empty(m, n, dtype=TYPES[case["out"]], device="cuda")}


def _data(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"norm": _norm_data, "cache": _cache_data, "attend": _cache_data, "vec": _vec_data}[case["op"]](case, g)
    st["case"] = case
    return st


class _Held:
    """A weight on the backend, freed with the state that holds it."""

    def __init__(self, weight):
        self.weight = weight

    def __del__(self):
        self.weight.free()


def _handles(st):
    """The handles and descriptions that a program keeps."""
    case = st["case"]
    mod, be = _framework()
    if case["op"] == "norm":
        st["rope"] = be.rope(case["dim"], _sections(case), neighbours=case["pairing"] == "neighbours", deal=case["deal"],
                             restart=case["restart"], base=case["base"])
        x, hq, hk = st["x"], case["q_heads"], case["k_heads"]
        nb = x.stride()[:2]
        st["sets"] = [mod.NormHeads(part.data_ptr(), heads, st[name + "_weight"].data_ptr(), st[name + "_out"].data_ptr(),
                                    bias=None if st[name + "_bias"] is None else st[name + "_bias"].data_ptr(), x_nb=nb)
                      for name, part, heads in (("q", x, hq), ("k", x[:, hq:], hk))]
    elif case["op"] == "vec":
        kind = mod.TYPE_Q4_0 if case["weights"] == "q4_0" else mod.TYPE_Q4_1
        torch.cuda.current_stream().synchronize()
        st["held"] = _Held(be.weight(kind, st.pop("blocks").data_ptr(), case["k"], case["n"]))
    else:
        st["cache"] = mod.KV4Cache(st["k_codes"].data_ptr(), st["v_codes"].data_ptr(), st["k_scale"].data_ptr(),
                                   st["v_scale"].data_ptr(), *st["k_codes"].shape[:3], case["dim"])
        new, total, width = st["new"], st["total"], st["table"].shape[1]
        st["batch"] = mod.KVBatch(st["table"].data_ptr(), width, st["row_start"].data_ptr(), st["kv_len"].data_ptr(), len(new),
                                  sum(new), max(new), max(total))
        if case["op"] == "cache":
            read = st["read"]
            st["batch_read"] = mod.KVBatch(st["table"].data_ptr(), width, st["read_start"].data_ptr(), st["kv_len"].data_ptr(),
                                           len(new), sum(read), max(read), max(total))
        else:
            st["attend"] = _kept["attend"]


def prepare(case, seed):
    if own:
        _framework()
        torch.cuda.set_stream(_kept["stream"])
    st = _data(case, seed)
    if own:
        _handles(st)
    return st


# ---- plain forms -----------------------------------------------------------------------------------------------


def _axis_and_index(case):
    """The axis of each pair, and the pair's place in its axis."""
    left, axis, place = _sections(case), [], []
    total, a = list(left), 0
    for _ in range(sum(left)):
        while not left[a % len(left)]:
            a += 1
        axis.append(a % len(left))
        place.append(total[a % len(left)] - left[a % len(left)])
        left[a % len(left)] -= 1
        a += 1 if case["deal"] else 0
    return axis, place


def _plain_norm(st):
    case, hq = st["case"], st["case"]["q_heads"]
    axis, place = _axis_and_index(case)
    n = len(axis)
    sections = _sections(case)
    power = [p / sections[a] if case["restart"] else i / n for i, (a, p) in enumerate(zip(axis, place))]
    freq = torch.pow(torch.tensor(case["base"], dtype=torch.float64, device="cuda"), -torch.tensor(power, dtype=torch.float64, device="cuda"))
    angle = st["pos"].double()[torch.tensor(axis, device="cuda")].t() * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    for name, x in (("q", st["x"][:, :hq]), ("k", st["x"][:, hq:hq + case["k_heads"]])):
        y = x.float()
        if case["kind"] == "layer":
            y = y - y.mean(-1, keepdim=True)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * st[name + "_weight"]
        if case["kind"] == "layer":
            y = y + st[name + "_bias"]
        if case["pairing"] == "halves":
            a, b = y[..., :n], y[..., n:2 * n]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        st[name + "_out"].copy_(torch.cat([turned, y[..., 2 * n:]], -1))
    return st["q_out"], st["k_out"]


def _split4(codes):
    """uint8 [..., d / 2] -> whole numbers -8 .. 7 [..., d]."""
    return torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(torch.int8) - 8


def _plain_write(st, name):
    """The rows of st[name] into the cache."""
    x, p, start = st[name], st["case"]["page"], st["row_start"].long()
    count = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=x.shape[0])
    pos = torch.arange(x.shape[0], device="cuda") - start[seq] + (st["kv_len"].long() - count)[seq]
    page = st["table"].long()[seq, pos // p]
    y = x.float().unflatten(-1, (-1, 32))
    high, low = y.amax(-1, keepdim=True), y.amin(-1, keepdim=True)
    top = torch.where(high >= -low, high, low)
    scale = torch.where(top.abs() < SMALL, 0.0, top / -8).bfloat16()
    by = scale.double()
    code = torch.where(by != 0, y.double() / torch.where(by != 0, by, 1.0), 0.0).round().clamp(-8, 7).to(torch.int16).flatten(-2) + 8
    st[name + "_codes"][page, :, pos % p] = (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8)
    st[name + "_scale"][page, :, pos % p] = scale[..., 0]


def _plain_read(st, name):
    p, out, start = st["case"]["page"], st[name + "_out"], st["read_start"].long()
    count = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=out.shape[0])
    pos = torch.arange(out.shape[0], device="cuda") - start[seq] + (st["kv_len"].long() - count)[seq]
    page = st["table"].long()[seq, pos // p]
    code, scale = _split4(st[name + "_codes"][page, :, pos % p]), st[name + "_scale"][page, :, pos % p]
    out.copy_((code.unflatten(-1, (-1, 32)).float() * scale.float()[..., None]).flatten(-2))
    return out


def _plain_attend(st):
    case, q = st["case"], st["q"]
    new, total, p, group = st["new"], st["total"], case["page"], case["heads"] // case["kv_heads"]
    seqs, most_q, used = len(new), max(new), -(-max(total) // p)
    heads, d = case["kv_heads"], case["dim"]
    start, end = st["row_start"].long(), st["kv_len"].long()
    count = start[1:] - start[:-1]
    at = torch.arange(most_q, device="cuda")
    rows = (start[:-1, None] + at).clamp(max=q.shape[0] - 1)
    page = st["table"].long()[:, :used].flatten()

    def whole(name):  # [seqs, heads, used * p, d]
        x = _split4(st[name + "_codes"][page]).unflatten(-1, (-1, 32)).float() * st[name + "_scale"][page].float()[..., None]
        return x.view(seqs, used, heads, p, d).transpose(1, 2).reshape(seqs, heads, used * p, d)

    qs = q[rows].float().view(seqs, most_q, heads, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, heads, group * most_q, d)
    score = (qs @ whole("k").transpose(2, 3)).mul_(st["scale"]).view(seqs, heads, group, most_q, used * p)
    key = torch.arange(used * p, device="cuda")
    last = (end - count)[:, None] + at if case["causal"] else (end - 1)[:, None].expand(seqs, most_q)
    seen = key <= last[..., None]
    if case["window"]:
        seen &= key > last[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    w = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    norm = w.sum(-1, keepdim=True).clamp(min=1e-30)
    y = (w.view(seqs, heads, group * most_q, used * p) @ whole("v")).view(seqs, heads, group, most_q, d) / norm
    y = y.permute(0, 3, 1, 2, 4).reshape(seqs, most_q, heads * group, d)
    st["out"].copy_(y[at[None] < count[:, None]])
    return st["out"]


def _plain_vec(st):
    case, blocks = st["case"], st["blocks"]
    head = 2 if case["weights"] == "q4_0" else 4
    half = blocks[:, :head].contiguous().view(torch.float16).float()
    packed = blocks[:, head:]
    code = torch.cat([packed & 15, packed >> 4], 1).float()
    w = (code - 8) * half if case["weights"] == "q4_0" else code * half[:, :1] + half[:, 1:]
    y = st["x"].float() @ w.view(case["n"], case["k"]).t()
    if st["bias"] is not None:
        y = y + st["bias"]
    st["out"].copy_(y)
    return st["out"]


# ---- one pass --------------------------------------------------------------------------------------------------


def _calls(st):
    case = st["case"]
    mod, be = _framework()
    types = {torch.float32: mod.TYPE_F32, torch.float16: mod.TYPE_F16, torch.bfloat16: mod.TYPE_BF16}
    if case["op"] == "norm":
        st["rope"].norm(st["sets"], types[st["x"].dtype], st["pos"].data_ptr(), st["x"].shape[0], types[st["q_out"].dtype],
                        eps=st["eps"], layer=case["kind"] == "layer")
        return st["q_out"], st["k_out"]
    if case["op"] == "vec":
        x, out, bias = st["x"], st["out"], st["bias"]
        be.mul_mat_vec(st["held"].weight, x.data_ptr(), types[x.dtype], x.shape[0], out.data_ptr(), types[out.dtype],
                       bias=None if bias is None else bias.data_ptr())
        return out
    if case["op"] == "cache":
        k, v, k_out, v_out = st["k"], st["v"], st["k_out"], st["v_out"]
        be.kv4_write(st["cache"], st["batch"], types[k.dtype], k.data_ptr(), v.data_ptr())
        be.kv4_read(st["cache"], st["batch_read"], types[k.dtype], k_out.data_ptr(), v_out.data_ptr())
        return k_out, v_out
    q, out = st["q"], st["out"]
    st["attend"].run(st["cache"], st["batch"], types[q.dtype], q.data_ptr(), q.shape[1], out.data_ptr(),
                     scale=st["scale"], causal=case["causal"], window=case["window"])
    return out


def run(state):
    st, case = state, state["case"]
    if own:
        there = _kept["stream"]
        here = torch.cuda.current_stream(there.device_index)
        if here.cuda_stream == there.cuda_stream:
            return _calls(st)
        there.wait_stream(here)
        result = _calls(st)
        here.wait_stream(there)
        return result
    if case["op"] == "norm":
        return _plain_norm(st)
    if case["op"] == "vec":
        return _plain_vec(st)
    if case["op"] == "cache":
        _plain_write(st, "k")
        _plain_write(st, "v")
        return _plain_read(st, "k"), _plain_read(st, "v")
    return _plain_attend(st)


def _seen(case, new, total):
    """(query, key) pairs that are not masked, and keys that some query sees, over the sequences."""
    pairs = keys = 0
    for n, t in zip(new, total):
        if not case["causal"]:
            pairs, keys = pairs + n * t, keys + t
            continue
        w = case["window"] or t
        pairs += sum(min(t - n + i + 1, w) for i in range(n))
        keys += min(t, n + w - 1)
    return pairs, keys


def work(case):
    if case["op"] == "norm":
        values = _tokens(case) * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": values * (BYTES[case["type"]] + BYTES[case["out"]]) + 4 * len(_sections(case)) * _tokens(case),
                "flops": values * (4 if case["kind"] == "rms" else 7)
                + 6 * _tokens(case) * (case["q_heads"] + case["k_heads"]) * sum(_sections(case))}
    if case["op"] == "vec":
        m, k, n = case["rows"], case["k"], case["n"]
        block = 18 if case["weights"] == "q4_0" else 20
        return {"bytes": n * (k // 32) * block + m * k * BYTES[case["type"]] + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0),
                "flops": 2 * m * k * n}
    new, past = _lengths(case)
    total = [a + b for a, b in zip(new, past)]
    p, heads, d = case["page"], case["kv_heads"], case["dim"]
    held = d // 2 + d // 16  # bytes of a token's head
    if case["op"] == "cache":
        # the new rows in, their codes and scales out; those of the tokens read back in, their values out
        read = [t if case["read"] == "all" else t - (b // p) * p for t, b in zip(total, past)]
        return {"bytes": 2 * heads * (sum(new) + sum(read)) * (d * BYTES[case["type"]] + held),
                "flops": 2 * heads * d * (4 * sum(new) + sum(read))}
    pairs, keys = _seen(case, new, total)
    return {"bytes": 2 * keys * heads * held + 2 * 2 * sum(new) * case["heads"] * d, "flops": 4 * pairs * case["heads"] * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def _exact_norm(case, st):
    sections = _sections(case)
    n, queue = sum(sections), []
    if case["deal"]:  # one pair to each axis in turn, while it has any left
        for turn in range(max(sections)):
            queue += [(a, turn) for a in range(len(sections)) if turn < sections[a]]
    else:
        queue = [(a, j) for a in range(len(sections)) for j in range(sections[a])]
    result = []
    for name, first, heads in (("q", 0, case["q_heads"]), ("k", case["q_heads"], case["k_heads"])):
        x = st["x"].double()[:, first:first + heads]
        if case["kind"] == "layer":
            center = x - x.sum(-1, keepdim=True) / case["dim"]
            x = center / torch.sqrt(center.pow(2).sum(-1, keepdim=True) / case["dim"] + st["eps"]) * st[name + "_weight"].double()
            x = x + st[name + "_bias"].double()
        else:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["dim"] + st["eps"]) * st[name + "_weight"].double()
        y = x.clone()
        for i, (a, j) in enumerate(queue):
            w = math.exp(-math.log(case["base"]) * (j / sections[a] if case["restart"] else i / n))
            turn = torch.polar(torch.ones_like(st["pos"][a], dtype=torch.float64), st["pos"][a].double() * w)[:, None]
            d0, d1 = (i, i + n) if case["pairing"] == "halves" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., d0], x[..., d1]) * turn
            y[..., d0], y[..., d1] = z.real, z.imag
        result.append(y)
    return tuple(result)


def _values(codes, scale):
    """float64 of uint8 codes [..., d / 2] and their scales [..., d / 32]."""
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    out[..., 0::2] = (codes % 16).double() - 8
    out[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double() - 8
    return out * scale.double().repeat_interleave(32, -1)


def _exact_cache(case, st, name):
    p, rows, out, at = case["page"], st[name].double(), [], 0
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        pages = st["table"][s, :-(-t // p)].long()
        whole = _values(st[name + "_codes"][pages], st[name + "_scale"][pages]).transpose(1, 2).flatten(0, 1)[:t]
        x = rows[at:at + n].reshape(n, case["kv_heads"], -1, 32)
        at += n
        most = x.abs().amax(-1, keepdim=True)
        sign = torch.where((x == most).any(-1, keepdim=True), -1.0, 1.0).double()
        unit = (sign * most / 8).to(torch.bfloat16).double() * (most >= SMALL)  # scales are held in bf16
        code = torch.nan_to_num((x / unit).round(), nan=0.0).clamp(-8, 7)
        whole[t - n:] = (code * unit).flatten(-2)
        out.append(whole[t - st["read"][s]:])
    return torch.cat(out)


def _exact_attend(case, st):
    p, group, out, at = case["page"], case["heads"] // case["kv_heads"], [], 0
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        pages = st["table"][s, :-(-t // p)].long()
        k, v = (_values(st[c + "_codes"][pages], st[c + "_scale"][pages]).transpose(0, 1).flatten(1, 2)[:, :t] for c in ("k", "v"))
        q = st["q"][at:at + n].double()
        at += n
        place = torch.arange(t - n, t, device="cuda")[:, None] if case["causal"] else torch.full((n, 1), t - 1, device="cuda")
        gap = place - torch.arange(t, device="cuda")
        hidden = (gap < 0) | (gap >= case["window"]) if case["window"] else gap < 0
        heads = []
        for h in range(case["heads"]):
            z = (q[:, h] @ k[h // group].t()) * st["scale"]
            heads.append(torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[h // group])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _exact_vec(case, st):
    head = {"q4_0": 2, "q4_1": 4}[case["weights"]]
    x, out, each = st["x"].double().t().contiguous(), [], 4096
    for first in range(0, case["n"], each):  # rows of the weights at a time
        raw = st["blocks"][first * (case["k"] // 32):(first + each) * (case["k"] // 32)]
        d = raw[:, :2].contiguous().view(torch.float16).double()
        low = raw[:, 2:4].contiguous().view(torch.float16).double() if head == 4 else -8 * d
        w = torch.empty(raw.shape[0], 32, dtype=torch.float64, device=raw.device)
        w[:, :16] = (raw[:, head:] % 16).double() * d + low
        w[:, 16:] = torch.div(raw[:, head:], 16, rounding_mode="floor").double() * d + low
        out.append((w.view(-1, case["k"]) @ x).t())
    y = torch.cat(out, 1)
    return y if st["bias"] is None else y + st["bias"].double()


def exact(case, seed):
    st = _data(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, st)
    if case["op"] == "cache":
        return _exact_cache(case, st, "k"), _exact_cache(case, st, "v")
    if case["op"] == "vec":
        return _exact_vec(case, st)
    return _exact_attend(case, st)
