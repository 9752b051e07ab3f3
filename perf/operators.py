"""Measured cases of the sequence-cache operators: the rotation by positions of several axes, the 8-bit paged
key/value cache as it is written and read back, and the attention over it.

listed() and draw() give the cases, prepare() a program's data on the GPU, run() one pass through an operator:
in its plain form (elementary torch operations) where `own` is false, by the library's calls where it is true.
exact() is the operators' definition in 64 bits.

The backend launches on a stream of its own, which waits for no other.  A program that makes its inputs with torch
makes that stream torch's current one, as prepare() does, and everything is in order; where another stream is current
when run() is called, the two wait for each other around the calls.  Results are ready on the current stream.

The cache: codes int8 [pages][kv heads][page tokens][head dim] and one f32 scale for each page and kv head, for
keys and for values.  A sequence's tokens [i P, (i + 1) P) lie in the page that entry i of its row of the block
table names.  A batch gives each sequence a run of rows (row_start) and its length with these rows (kv_len): its
rows are its last tokens.  Writing rows into a page takes the scale max(old scale, amax / 127), the old one where
the page held tokens before; the older codes are rounded again to it.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SMALL = 2.0 ** -100  # pages whose largest value is below this hold zeros

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
    rope = dict(op="rope", sections="", pairing="halves", deal=False, restart=False, base=1e6, first=0, text=0)
    cache = dict(op="cache", kv_heads=8, dim=128, page=64, type="bf16")
    attend = dict(op="attend", heads=32, kv_heads=8, dim=128, page=64, type="bf16", causal=True, window=0)
    return [
        # one step of 7 sequences far into a conversation about a video: queries and keys of one token each
        dict(rope, name="rope_step", text=7, frames=0, height=0, width=0, heads=40, dim=128, sections="24,20,20", deal=True,
             base=5e6, first=200000, type="bf16", out="bf16"),
        # the 72 x 72 tokens of one image in the encoder's global blocks: two axes, frequencies of their own, f32 -> f16
        dict(rope, name="rope_image", frames=1, height=72, width=72, heads=32, dim=64, sections="0,16,16", pairing="neighbours",
             restart=True, base=1e4, type="f32", out="f16"),
        # a video prompt of 9 frames between text
        dict(rope, name="rope_video", text=301, frames=9, height=36, width=64, heads=40, dim=128, sections="16,24,24",
             first=1000, type="bf16", out="bf16"),
        # every sequence of a serving batch appends one token, its last page is read back
        dict(cache, name="cache_step", seqs=64, new=1, new_max=1, past=100, past_max=4000, read="page"),
        # ragged prompts appended behind earlier ones, the whole contexts read back
        dict(cache, name="cache_prompt", seqs=5, new=900, new_max=4500, past=0, past_max=1500, page=16, type="f16", read="all"),
        # a single token of a single short sequence: latency
        dict(attend, name="attend_one", seqs=1, new=1, new_max=1, past=700, past_max=700),
        # a serving batch, one token each, ragged lengths
        dict(attend, name="attend_batch", seqs=64, new=1, new_max=1, past=500, past_max=8100),
        # two long contexts, one token each, heads without groups
        dict(attend, name="attend_long", seqs=2, new=1, new_max=1, past=100000, past_max=131000, heads=8, kv_heads=8, page=128,
             type="f16"),
        # several drafted tokens of each sequence at once
        dict(attend, name="attend_few", seqs=16, new=3, new_max=6, past=900, past_max=6000, heads=24, kv_heads=8, page=16),
        # parts of prompts behind earlier contexts, with a sliding window
        dict(attend, name="attend_chunk", seqs=4, new=129, new_max=700, past=1000, past_max=7000, kv_heads=4, page=32, type="f16",
             window=2000),
        # a whole prompt of one sequence
        dict(attend, name="attend_prompt", seqs=1, new=4096, new_max=4096, past=0, past_max=0),
        # an image's 72 x 72 tokens attend to two cached images: no mask, no groups, the encoder's heads
        dict(attend, name="attend_images", seqs=1, new=5184, new_max=5184, past=5184, past_max=5184, heads=16, kv_heads=16, dim=64,
             causal=False, type="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["rope", "cache", "attend", "attend"])
    dim = rng.choice([64, 128, 128])
    if op == "rope":
        pairs = dim // 2
        axes = rng.choice([1, 2, 3, 3, 4])
        cut = sorted(rng.randint(1, pairs - 1) for _ in range(axes - 1))
        sections = [b - a for a, b in zip([0] + cut, cut + [pairs])]
        if rng.random() < 0.3:  # a part of each head is not turned
            sections[-1] = (sections[-1] + 1) // 2
        text, frames = _log_int(rng, 1, 2000), rng.choice([0, 1, rng.randint(2, 6)])
        height, width = rng.randint(5, 36), rng.randint(5, 48)
        return dict(op="rope", text=text, frames=frames, height=height, width=width, heads=rng.randint(1, 40), dim=dim,
                    sections=",".join(map(str, sections)), pairing=rng.choice(["halves", "neighbours"]), deal=rng.random() < 0.5,
                    restart=rng.random() < 0.3, base=rng.choice([1e4, 5e5, 1e6]), first=rng.choice([0, _log_int(rng, 10, 1000000)]),
                    type=rng.choice(["bf16", "f16", "f32"]), out=rng.choice(["bf16", "f16", "f32"]))
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
        past_max = _log_int(rng, 60, min(100000, 400000 // seqs))
    elif kind == "few":
        seqs, new, new_max = _log_int(rng, 1, 24), 2, rng.randint(3, 9)
        past_max = _log_int(rng, 60, min(30000, 150000 // seqs))
    elif kind == "prompt":
        seqs = rng.randint(1, 4)
        new = _log_int(rng, 20, 2500 // seqs)
        new_max, past_max = min(2800, new + new // 2 + 1), _log_int(rng, 1, 2500)
    else:
        seqs, new = rng.randint(1, 2), _log_int(rng, 10, 2500)
        new_max, past_max, window = new + 7, _log_int(rng, 100, 2500), 0
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


def _prepare_rope(case, g):
    """Half of the text, the frames' grid, the rest of the text: positions as a prompt with a video has them."""
    sections, n = _sections(case), _tokens(case)
    before = case["text"] // 2
    f, h, w = case["frames"], case["height"], case["width"]
    lead = torch.arange(before).expand(4, before)
    grid = torch.stack([x.reshape(-1) for x in torch.meshgrid(torch.arange(f), torch.arange(h), torch.arange(w), indexing="ij")])
    grid = torch.cat([grid, grid[:1]]) + before
    rest = torch.arange(case["text"] - before).expand(4, -1) + (before + max(f, h, w) if f else before)
    pos = torch.cat([lead, grid, rest], 1)[: len(sections)] + case["first"]
    x = torch.randn(n, case["heads"], case["dim"], generator=g, device="cuda").to(TYPES[case["type"]])
    return {"x": x, "pos": pos.to(torch.int32).contiguous().cuda(), "out": torch.empty(x.shape, dtype=TYPES[case["out"]], device="cuda")}


def _prepare_cache(case, g):
    new, past = _lengths(case)
    H, D, P, t = case["kv_heads"], case["dim"], case["page"], TYPES[case["type"]]
    total = [a + b for a, b in zip(new, past)]
    used = [-(-n // P) for n in total]
    width = max(used) + 1
    pages = sum(used) + 3
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
        st[name + "_codes"] = torch.randint(-127, 128, (pages, H, P, D), generator=g, device="cuda", dtype=torch.int8)
        st[name + "_scale"] = torch.exp(0.3 * torch.randn(pages, H, generator=g, device="cuda")) * (0.025 if name == "k" else 0.02)
    if case["op"] == "cache":
        rows = sum(new)
        read = [n if case["read"] == "all" else n - (b // P) * P for n, b in zip(total, past)]
        st["read"] = read
        st["read_start"] = torch.tensor(_starts(read), dtype=torch.int32, device="cuda")
        for name in ("k", "v"):
            # channels of keys differ in size
            size = torch.exp(0.6 * torch.randn(H, D, generator=g, device="cuda")) if name == "k" else 1.0
            st[name] = (torch.randn(rows, H, D, generator=g, device="cuda") * size).to(t)
            st[name + "_out"] = torch.empty(sum(read), H, D, dtype=t, device="cuda")
    else:
        # queries of the size that spreads the softmax over some tens of keys
        st["q"] = (torch.randn(sum(new), case["heads"], D, generator=g, device="cuda") * 1.2).to(t)
        st["out"] = torch.empty_like(st["q"])
        st["scale"] = 1.0 / math.sqrt(D)
    return st


def prepare(case, seed):
    if own:
        _framework()
        torch.cuda.set_stream(_kept["stream"])
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = _prepare_rope(case, g) if case["op"] == "rope" else _prepare_cache(case, g)
    st["case"] = case
    if own:  # the handles and descriptions that a program keeps
        mod, be = _framework()
        if case["op"] == "rope":
            st["rope"] = be.rope(case["dim"], _sections(case), neighbours=case["pairing"] == "neighbours", deal=case["deal"],
                                 restart=case["restart"], base=case["base"])
        else:
            st["cache"] = mod.KVCache(st["k_codes"].data_ptr(), st["v_codes"].data_ptr(), st["k_scale"].data_ptr(),
                                      st["v_scale"].data_ptr(), *st["k_codes"].shape)
            st["batch"] = mod.KVBatch(st["table"].data_ptr(), st["table"].shape[1], st["row_start"].data_ptr(),
                                      st["kv_len"].data_ptr(), len(st["new"]), sum(st["new"]), max(st["new"]), max(st["total"]))
            if case["op"] == "cache":
                st["batch_read"] = mod.KVBatch(st["table"].data_ptr(), st["table"].shape[1], st["read_start"].data_ptr(),
                                               st["kv_len"].data_ptr(), len(st["new"]), sum(st["read"]), max(st["read"]),
                                               max(st["total"]))
            else:
                st["attend"] = _kept["attend"]
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


def _plain_rope(st):
    case, x = st["case"], st["x"]
    axis, place = _axis_and_index(case)
    n = len(axis)
    sections = _sections(case)
    power = [p / sections[a] if case["restart"] else i / n for i, (a, p) in enumerate(zip(axis, place))]
    freq = torch.pow(torch.tensor(case["base"], dtype=torch.float64, device="cuda"), -torch.tensor(power, dtype=torch.float64, device="cuda"))
    angle = st["pos"].double()[torch.tensor(axis, device="cuda")].t() * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    y = x.float()
    if case["pairing"] == "halves":
        a, b = y[..., :n], y[..., n:2 * n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    st["out"].copy_(torch.cat([turned, y[..., 2 * n:]], -1))
    return st["out"]


def _plain_write(st, name):
    """The rows of st[name] into the pages of the cache, all pages that they touch at once."""
    codes, scale, x, P = st[name + "_codes"], st[name + "_scale"], st[name], st["case"]["page"]
    new, total = st["new"], st["total"]
    touched = max((t - 1) // P - (t - n) // P + 1 for n, t in zip(new, total))
    end = st["kv_len"].long()
    row0 = st["row_start"].long()
    begin = end - (row0[1:] - row0[:-1])
    index = (begin // P)[:, None] + torch.arange(touched, device="cuda")
    live = index * P < end[:, None]
    page = st["table"].long().gather(1, index.clamp(max=st["table"].shape[1] - 1))[live]
    pos = (index[:, :, None] * P + torch.arange(P, device="cuda"))[live]
    seq = torch.arange(len(new), device="cuda")[:, None].expand_as(index)[live]
    fresh = ((pos >= begin[seq][:, None]) & (pos < end[seq][:, None]))[:, None, :, None]
    old = (pos < begin[seq][:, None])[:, None, :, None]
    rows = x[(row0[seq][:, None] + pos - begin[seq][:, None]).clamp(0, x.shape[0] - 1)].transpose(1, 2).float()
    amax = torch.where(fresh, rows.abs(), 0.0).amax((2, 3))
    held = torch.where((pos[:, :1] < begin[seq][:, None]), scale[page], 0.0)
    wide = torch.maximum(held, torch.where(amax < SMALL, 0.0, amax / 127.0))
    to = torch.where(wide > 0, wide, 1.0).double()[:, :, None, None]
    put = (rows.double() / to).round().clamp(-127, 127)
    again = (codes[page].double() * held.double()[:, :, None, None] / to).round()
    codes[page] = torch.where(fresh, put, torch.where(old, again, codes[page].double())).to(torch.int8)
    scale[page] = wide


def _plain_read(st, name):
    codes, scale, P, out = st[name + "_codes"], st[name + "_scale"], st["case"]["page"], st[name + "_out"]
    start = st["read_start"].long()
    count = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(len(count), device="cuda"), count, output_size=out.shape[0])
    pos = torch.arange(out.shape[0], device="cuda") - start[seq] + (st["kv_len"].long() - count)[seq]
    page = st["table"].long()[seq, pos // P]
    out.copy_(codes[page, :, pos % P].float() * scale[page][:, :, None])
    return out


def _plain_attend(st):
    case, q = st["case"], st["q"]
    new, total, P, G = st["new"], st["total"], case["page"], case["heads"] // case["kv_heads"]
    S, most_q, used = len(new), max(new), -(-max(total) // P)
    H, D = case["kv_heads"], case["dim"]
    start, end = st["row_start"].long(), st["kv_len"].long()
    count = start[1:] - start[:-1]
    at = torch.arange(most_q, device="cuda")
    rows = (start[:-1, None] + at).clamp(max=q.shape[0] - 1)
    page = st["table"].long()[:, :used].flatten()

    def whole(name):  # [S, H, used * P, D]
        x = st[name + "_codes"][page].float() * st[name + "_scale"][page][:, :, None, None]
        return x.view(S, used, H, P, D).transpose(1, 2).reshape(S, H, used * P, D)

    qs = q[rows].float().view(S, most_q, H, G, D).permute(0, 2, 3, 1, 4).reshape(S, H, G * most_q, D)
    score = (qs @ whole("k").transpose(2, 3)).mul_(st["scale"]).view(S, H, G, most_q, used * P)
    key = torch.arange(used * P, device="cuda")
    last = (end - count)[:, None] + at if case["causal"] else (end - 1)[:, None].expand(S, most_q)
    seen = key <= last[..., None]
    if case["window"]:
        seen &= key > last[..., None] - case["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    p = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    norm = p.sum(-1, keepdim=True).clamp(min=1e-30)
    y = (p.view(S, H, G * most_q, used * P) @ whole("v")).view(S, H, G, most_q, D) / norm
    y = y.permute(0, 3, 1, 2, 4).reshape(S, most_q, H * G, D)
    st["out"].copy_(y[at[None] < count[:, None]])
    return st["out"]


# ---- one pass --------------------------------------------------------------------------------------------------


def _calls(st):
    case = st["case"]
    mod, be = _framework()
    types = {torch.float32: mod.TYPE_F32, torch.float16: mod.TYPE_F16, torch.bfloat16: mod.TYPE_BF16}
    if case["op"] == "rope":
        x, out = st["x"], st["out"]
        st["rope"].apply(x.data_ptr(), types[x.dtype], st["pos"].data_ptr(), x.shape[0], x.shape[1], out.data_ptr(),
                         types[out.dtype])
        return out
    if case["op"] == "cache":
        k, v, k_out, v_out = st["k"], st["v"], st["k_out"], st["v_out"]
        be.kv_write(st["cache"], st["batch"], types[k.dtype], k.data_ptr(), v.data_ptr())
        be.kv_read(st["cache"], st["batch_read"], types[k.dtype], k_out.data_ptr(), v_out.data_ptr())
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
    if case["op"] == "rope":
        return _plain_rope(st)
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
    size = {"f32": 4, "f16": 2, "bf16": 2}
    D = case["dim"]
    if case["op"] == "rope":
        values, n = _tokens(case) * case["heads"] * D, len(_sections(case))
        return {"bytes": values * (size[case["type"]] + size[case["out"]]) + 4 * n * _tokens(case),
                "flops": 6 * _tokens(case) * case["heads"] * sum(_sections(case))}
    new, past = _lengths(case)
    total = [a + b for a, b in zip(new, past)]
    P, H = case["page"], case["kv_heads"]
    if case["op"] == "cache":
        # the new rows in, their codes out; the codes of the tokens read back in, their values out
        read = [t if case["read"] == "all" else t - (b // P) * P for t, b in zip(total, past)]
        values, back = sum(new) * H * D, sum(read) * H * D
        return {"bytes": 2 * (values * (size[case["type"]] + 1) + back * (size[case["type"]] + 1)), "flops": 2 * (3 * values + back)}
    pairs, keys = _seen(case, new, total)
    return {"bytes": 2 * keys * H * D + 2 * 2 * sum(new) * case["heads"] * D + 8 * (keys // P) * H,
            "flops": 4 * pairs * case["heads"] * D}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------


def _exact_rope(case, st):
    sections = _sections(case)
    n, queue = sum(sections), []
    if case["deal"]:  # one pair to each axis in turn, while it has any left
        for turn in range(max(sections)):
            queue += [(a, turn) for a in range(len(sections)) if turn < sections[a]]
    else:
        queue = [(a, j) for a in range(len(sections)) for j in range(sections[a])]
    x = st["x"].double()
    y = x.clone()
    for i, (a, j) in enumerate(queue):
        w = math.exp(-math.log(case["base"]) * (j / sections[a] if case["restart"] else i / n))
        turn = torch.polar(torch.ones_like(st["pos"][a], dtype=torch.float64), st["pos"][a].double() * w)[:, None]
        d0, d1 = (i, i + n) if case["pairing"] == "halves" else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., d0], x[..., d1]) * turn
        y[..., d0], y[..., d1] = z.real, z.imag
    return y


def _exact_cache(case, st, name):
    P, codes, scale = case["page"], st[name + "_codes"].double(), st[name + "_scale"].double()
    rows, out, at = st[name].double(), [], 0
    table = st["table"].tolist()
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        b = t - n
        for i in range(b // P, -(-t // P)):
            page, lo, hi = table[s][i], max(b, i * P), min(t, (i + 1) * P)
            x = rows[at + lo - b:at + hi - b].transpose(0, 1)
            most = x.abs().amax((1, 2))
            unit = (most.float() / 127).double() * (most >= SMALL)  # scales are held in 32 bits
            if lo > i * P:
                unit = torch.maximum(unit, scale[page])
                codes[page, :, :lo - i * P] = (codes[page, :, :lo - i * P] * (scale[page] / unit)[:, None, None]).round()
            codes[page, :, lo - i * P:hi - i * P] = (x / unit[:, None, None]).round()
            scale[page] = unit
        at += n
        first = t - st["read"][s]
        for i in range(first // P, -(-t // P)):
            lo, hi = max(first, i * P), min(t, (i + 1) * P)
            out.append((codes[table[s][i], :, lo - i * P:hi - i * P] * scale[table[s][i]][:, None, None]).transpose(0, 1))
    return torch.cat(out)


def _exact_attend(case, st):
    P, G, out, at = case["page"], case["heads"] // case["kv_heads"], [], 0
    for s, (n, t) in enumerate(zip(st["new"], st["total"])):
        pages = st["table"][s, :-(-t // P)].long()
        k, v = ((st[c + "_codes"][pages].double() * st[c + "_scale"][pages].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :t]
                for c in ("k", "v"))
        q = st["q"][at:at + n].double()
        at += n
        place = torch.arange(t - n, t, device="cuda")[:, None] if case["causal"] else torch.full((n, 1), t - 1, device="cuda")
        gap = place - torch.arange(t, device="cuda")
        hidden = (gap < 0) | (gap >= case["window"]) if case["window"] else gap < 0
        heads = []
        for h in range(case["heads"]):
            z = (q[:, h] @ k[h // G].t()) * st["scale"]
            heads.append(torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v[h // G])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, st)
    if case["op"] == "cache":
        return _exact_cache(case, st, "k"), _exact_cache(case, st, "v")
    return _exact_attend(case, st)
