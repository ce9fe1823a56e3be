"""The sequence operators (rotary positions, the 8-bit paged cache and the attention over it): cases, their plain forms in
elementary torch operations, and the calls a user makes.

A cache holds, for each page of `page` tokens and each head, float8 (e4m3) codes and one power-of-two scale for the keys and
one for the values. Layout of the codes, in bytes:
    keys    [pages][heads][page/8][dim/16][8 tokens][16 dims]
    values  [pages][heads][page/16][dim][16 tokens]
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases


def listed():
    return [
        # q and k heads of one fused projection buffer, one decode step of 16 sequences deep into long inputs
        dict(name="rotary one token", op="rotary", rows=16, heads=40, dim=128, rot=128, dtype="bf16", axes=1, adjacent=False, inverse=False, far=900000),
        # a prompt batch whose tokens have three places: chain, residue, atom
        dict(name="rotary three axes", op="rotary", rows=8192, heads=40, dim=128, rot=128, dtype="bf16", axes=3, adjacent=False, inverse=False, far=8192),
        # gradients of a training step in 32 bits, neighbouring pairs, half of each head rotated, an odd number of rows
        dict(name="rotary gradient", op="rotary", rows=4099, heads=20, dim=64, rot=32, dtype="f32", axes=2, adjacent=True, inverse=True, far=100000),
        # one token for each of 64 sequences of up to 2048, queries rotated on the way
        dict(name="append one token", op="append", seqs=64, new=1, len=2048, ragged=True, q_heads=32, heads=8, dim=128, page=64, rot=128, dtype="bf16", axes=1, adjacent=False),
        # eight prompts of about a thousand tokens
        dict(name="append prompts", op="append", seqs=8, new=1024, len=1024, ragged=True, q_heads=32, heads=8, dim=128, page=64, rot=128, dtype="bf16", axes=1, adjacent=False),
        # the next pieces of three long inputs, small pages that begin half full, 20 heads of 64
        dict(name="append pieces", op="append", seqs=3, new=777, len=5003, ragged=True, q_heads=20, heads=20, dim=64, page=16, rot=64, dtype="f16", axes=2, adjacent=True),
        # a single short sequence, one token: latency
        dict(name="attention one short", op="attention", seqs=1, new=1, len=700, ragged=False, q_heads=32, heads=8, dim=128, page=16, dtype="bf16", causal=True, window=0, lse=False),
        # a full decode batch
        dict(name="attention one token", op="attention", seqs=64, new=1, len=8192, ragged=True, q_heads=32, heads=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=False),
        # one very long sequence on few heads: the keys have to be split
        dict(name="attention long", op="attention", seqs=1, new=1, len=200001, ragged=False, q_heads=16, heads=2, dim=128, page=128, dtype="bf16", causal=True, window=0, lse=True),
        # five guessed tokens verified at once, a head of keys for each head of queries
        dict(name="attention five tokens", op="attention", seqs=16, new=5, len=4096, ragged=True, q_heads=20, heads=20, dim=64, page=32, dtype="f16", causal=True, window=0, lse=False),
        # pieces of a thousand tokens against contexts of about eight thousand
        dict(name="attention pieces", op="attention", seqs=4, new=1024, len=8192, ragged=True, q_heads=32, heads=8, dim=128, page=64, dtype="bf16", causal=True, window=0, lse=True),
        # whole prompts with a window of a thousand tokens
        dict(name="attention window", op="attention", seqs=2, new=4096, len=4096, ragged=True, q_heads=16, heads=4, dim=64, page=64, dtype="f16", causal=True, window=1024, lse=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "attention", "attention"))
    if op == "rotary":
        dim = rng.choice((32, 48, 64, 80, 96, 128))
        rows, heads = _log(rng, 1, 8192), _log(rng, 1, 40)
        rot = dim if rng.random() < 0.6 else 2 * rng.randint(4, dim // 2)
        return dict(op=op, rows=rows, heads=heads, dim=dim, rot=rot, dtype=rng.choice(("bf16", "bf16", "f16", "f32")), axes=rng.randint(1, 4),
                    adjacent=rng.random() < 0.5, inverse=rng.random() < 0.4, far=_log(rng, 1, 1000000))
    dim, group = rng.choice((32, 64, 64, 96, 128, 128, 128)), rng.choice((1, 1, 2, 3, 4, 7, 8, 16))
    page = rng.choice((16, 32, 64, 64, 128))
    if op == "append":
        heads = _log(rng, 1, 20)
        seqs = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 8192 // seqs))
        length = new if rng.random() < 0.4 else new + _log(rng, 1, 4096)
        return dict(op=op, seqs=seqs, new=new, len=length, ragged=seqs > 1, q_heads=heads * min(group, 40 // heads), heads=heads, dim=dim, page=page,
                    rot=dim if rng.random() < 0.7 else dim // 2, dtype=rng.choice(("bf16", "bf16", "f16")), axes=rng.randint(1, 3), adjacent=rng.random() < 0.4)
    kind = rng.choice(("one", "one", "few", "many"))
    if kind == "many":
        heads, seqs = _log(rng, 1, 8), _log(rng, 1, 4)
        group = min(group, 4)
        new = _log(rng, 64, 4096 // seqs)
        length = new if rng.random() < 0.5 else new + _log(rng, 1, 4096)
        window = 0 if rng.random() < 0.7 else _log(rng, 16, 2048)
    else:
        heads = _log(rng, 1, 20)
        seqs = _log(rng, 1, 64)
        new = 1 if kind == "one" else rng.randint(2, 12)
        length = new + _log(rng, 1, max(64, min(200000, 64 * 8 * 8192 // (seqs * heads * 2))))
        window = 0 if rng.random() < 0.8 else _log(rng, 16, 4096)
    return dict(op=op, seqs=seqs, new=new, len=length, ragged=seqs > 1, q_heads=heads * group, heads=heads, dim=dim, page=page,
                dtype=rng.choice(("bf16", "bf16", "f16")), causal=rng.random() < 0.9, window=window, lse=rng.random() < 0.3)


def _counts(case):
    """(new rows, length with them) of every sequence: the case alone decides them."""
    rng = random.Random("%(seqs)d %(new)d %(len)d %(page)d" % case)
    if not case["ragged"]:
        return [case["new"]] * case["seqs"], [case["len"]] * case["seqs"]
    new, length = [], []
    for _ in range(case["seqs"]):
        n = 1 if case["new"] == 1 else rng.randint(max(1, (3 * case["new"]) // 4), case["new"])
        old = case["len"] - case["new"]
        new.append(n)
        length.append(n + (rng.randint(old // 2, old) if old else 0))
    return new, length


def _seen(case):
    """Pairs of a row and a key it sees."""
    total = 0
    for n, length in zip(*_counts(case)):
        for i in range(n):
            hi = length - n + i + 1 if case["causal"] else length
            lo = max(0, length - n + i + 1 - case["window"]) if case["window"] else 0
            total += max(0, hi - lo)
    return total


def _keys(case):
    """Keys that some row of a sequence sees, over the sequences."""
    return sum(min(length, case["window"] + n - 1) if case["window"] else length for n, length in zip(*_counts(case)))


def work(case):
    if case["op"] == "rotary":
        values = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2.0 * values * SIZE[case["dtype"]] + 4 * case["axes"] * case["rows"], "flops": 3.0 * values}
    rows = sum(_counts(case)[0])
    if case["op"] == "append":
        kv = rows * case["heads"] * case["dim"]
        q = rows * case["q_heads"] * case["dim"]
        return {"bytes": 2.0 * kv * (SIZE[case["dtype"]] + 1) + 2.0 * q * SIZE[case["dtype"]] + 4 * case["axes"] * rows, "flops": 6.0 * kv + 3.0 * q}
    io = 2.0 * rows * case["q_heads"] * case["dim"] * SIZE[case["dtype"]] + (4.0 * rows * case["q_heads"] if case["lse"] else 0)
    keys = _keys(case) * case["heads"] * (2.0 * case["dim"] + 8.0 / case["page"])
    return {"bytes": io + keys, "flops": 4.0 * _seen(case) * case["q_heads"] * case["dim"]}


# ---- inputs


def _sections(pairs, axes):
    return [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]


def _frequencies(pairs, axes):
    return torch.cat([10000.0 ** (-torch.arange(s, dtype=torch.float64) / max(1, s)) for s in _sections(pairs, axes)]).float().cuda()


def _quantised(values):
    """Codes and scales [..., 1, 1] of blocks [..., tokens, dims]: how a cache that was filled before looks."""
    top = values.abs().amax(dim=(-2, -1), keepdim=True)
    mantissa, exponent = torch.frexp(top)
    scale = torch.exp2((exponent - 9 + (mantissa > 0.875)).clamp(-40, 40).float())
    return (values / scale).to(torch.float8_e4m3fn), scale[..., 0, 0].contiguous()


def _key_layout(codes):
    n, h, p, d = codes.shape
    return codes.view(torch.uint8).view(n, h, p // 8, 8, d // 16, 16).permute(0, 1, 2, 4, 3, 5).contiguous().view(-1)


def _value_layout(codes):
    n, h, p, d = codes.shape
    return codes.view(torch.uint8).view(n, h, p // 16, 16, d).permute(0, 1, 2, 4, 3).contiguous().view(-1)


def _filled(case, pages, g):
    """A pool of pages as earlier tokens left it; a few of a head's channels are large, as they are in real keys."""
    h, p, d = case["heads"], case["page"], case["dim"]
    wide = 1 + 3 * (torch.rand(h, 1, d, device="cuda", generator=g) < 0.06).float()
    k, ks = _quantised(torch.randn(pages, h, p, d, device="cuda", generator=g) * wide)
    k = _key_layout(k)
    v, vs = _quantised(torch.randn(pages, h, p, d, device="cuda", generator=g) * torch.rand(h, 1, 1, device="cuda", generator=g).add(0.5))
    return dict(k=k, v=_value_layout(v), k_scale=ks, v_scale=vs)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]
    s = dict(case=case, sections=_sections(case["rot"] // 2, case["axes"]), freq=_frequencies(case["rot"] // 2, case["axes"])) if "rot" in case else dict(case=case)
    if case["op"] == "rotary":
        s["x"] = torch.randn(case["rows"], case["heads"], case["dim"], device="cuda", generator=g).to(t)
        s["y"] = torch.empty_like(s["x"])
        s["pos"] = torch.randint(0, case["far"], (case["axes"], case["rows"]), device="cuda", generator=g, dtype=torch.int32)
    else:
        new, length = _counts(case)
        rows, each = sum(new), [-(-n // case["page"]) for n in length]
        pages, wide = sum(each) + 3, max(each)
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table, at = torch.full((case["seqs"], wide), -1, dtype=torch.int32), 0
        fill = torch.arange(wide)[None, :] < torch.tensor(each)[:, None]
        table[fill] = torch.arange(sum(each), dtype=torch.int32)
        table = table.cuda()
        s["table"] = torch.where(table < 0, table, order[table.clamp(min=0).long()]).contiguous()
        s["first"] = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
        s["len"] = torch.tensor(length, dtype=torch.int32).cuda()
        s["max_new"], s["max_len"], s["pages"] = max(new), max(length), pages
        s.update(_filled(case, pages, g))
        s["q"] = torch.randn(rows, case["q_heads"], case["dim"], device="cuda", generator=g).to(t)
        s["out"] = torch.empty_like(s["q"])
        if case["op"] == "append":
            s["new_k"] = (1.5 * torch.randn(rows, case["heads"], case["dim"], device="cuda", generator=g)).to(t)
            s["new_v"] = torch.randn(rows, case["heads"], case["dim"], device="cuda", generator=g).to(t)
            i = torch.arange(rows, device="cuda")
            b = torch.searchsorted(s["first"][1:], i, right=True)
            place = (s["len"][b] - s["first"][b + 1] + i).to(torch.int32)
            s["pos"] = torch.stack([place // (7 ** a) for a in range(case["axes"])]).to(torch.int32).contiguous()
        else:
            s["lse"] = torch.empty(rows, case["q_heads"], device="cuda") if case["lse"] else None
    if own:
        s["plan"] = _plan(s)
    return s


# ---- the calls a user makes


def _plan(s):
    """The descriptors that a user's program keeps beside its buffers, and the attention's workspace."""
    import os
    import sys

    sys.path.insert(0, os.path.join(os.getcwd(), "colabfold-cuda-kernels_b200"))
    from colabfold_cuda_kernels import sequence as seq

    c = s["case"]
    rows = lambda x: seq.Rows(x.data_ptr(), c["dtype"], x.shape[1], x.stride(0), x.stride(1))  # noqa: E731
    p = dict(seq=seq)
    if "freq" in s:
        p["rotation"] = seq.Rotation(c["rot"], s["sections"], s["freq"].data_ptr(), s["pos"].data_ptr(), s["pos"].stride(0), adjacent=c["adjacent"])
    if c["op"] == "rotary":
        return dict(p, x=rows(s["x"]), y=rows(s["y"]))
    p["cache"] = seq.Cache(s["k"].data_ptr(), s["v"].data_ptr(), s["k_scale"].data_ptr(), s["v_scale"].data_ptr(), s["pages"], c["page"], c["heads"], c["dim"])
    p["batch"] = seq.Batch(c["seqs"], s["q"].shape[0], s["max_new"], s["max_len"], s["table"].shape[1], s["first"].data_ptr(), s["len"].data_ptr(), s["table"].data_ptr(),
                           s["table"].stride(0))
    p["q"], p["out"] = rows(s["q"]), rows(s["out"])
    if c["op"] == "append":
        p["k"], p["v"] = rows(s["new_k"]), rows(s["new_v"])
    else:
        need = seq.cache_attention_workspace_bytes(p["cache"], p["batch"], c["q_heads"])
        p["ws"], p["lse"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda"), s["lse"].data_ptr() if c["lse"] else 0
        p["ws_ptr"], p["ws_bytes"] = p["ws"].data_ptr(), need
    return p


def _own(s):
    c, p = s["case"], s["plan"]
    seq, stream = p["seq"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "rotary":
        seq.rotary(stream, p["rotation"], c["rows"], c["dim"], p["x"], p["y"], inverse=c["inverse"])
        return s["y"]
    if c["op"] == "append":
        seq.cache_append(stream, p["cache"], p["batch"], p["k"], p["v"], p["rotation"], p["q"], p["out"])
        return _appended(s, s["out"])
    seq.cache_attention(stream, p["cache"], p["batch"], p["q"], p["out"], c["dim"] ** -0.5, p["ws_ptr"], p["ws_bytes"], causal=c["causal"], window=c["window"], lse=p["lse"])
    return dict(out=s["out"], lse=s["lse"]) if c["lse"] else s["out"]


def _appended(s, q):
    return dict(q=q, k=s["k"].view(torch.float8_e4m3fn), v=s["v"].view(torch.float8_e4m3fn), k_scale=s["k_scale"], v_scale=s["v_scale"])


# ---- plain forms


def _rotated(s, x, inverse=False):
    """x [rows][heads][dim] with its first `rot` dims rotated, in 32 bits; the angles in 64."""
    c = s["case"]
    axis = torch.repeat_interleave(torch.arange(c["axes"], device="cuda"), torch.tensor(s["sections"], device="cuda"))
    angle = (s["pos"].double()[axis] * s["freq"].double()[:, None]).T[:, None, :]
    cos, sin = angle.cos().float(), angle.sin().float()
    sin = -sin if inverse else sin
    x, rot = x.float(), c["rot"]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if c["adjacent"] else (x[..., : rot // 2], x[..., rot // 2 : rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], dim=-1).flatten(-2) if c["adjacent"] else torch.cat([a, b], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _appended_block(s, rows, codes, scale, key):
    """New rows put into a copy of the touched blocks; what is older in them is brought to the new scale."""
    c = s["case"]
    n, h, p, d = s["pages"], c["heads"], c["page"], c["dim"]
    i = torch.arange(rows.shape[0], device="cuda")
    b = torch.searchsorted(s["first"][1:], i, right=True)
    place = (s["len"][b] - s["first"][b + 1] + i).long()
    old = (s["len"] - (s["first"][1:] - s["first"][:-1])).long()
    page, slot = s["table"][b, place // p].long(), place % p
    top = torch.zeros(n, h, device="cuda").scatter_reduce(0, page[:, None].expand(-1, h), rows.abs().amax(-1), "amax")
    mantissa, exponent = torch.frexp(top)
    want = torch.where(top > 0, exponent - 9 + (mantissa > 0.875), -40).clamp(-40, 40)
    half = old % p  # older rows in the block that a sequence's first new row falls into
    first_page = s["table"][torch.arange(c["seqs"], device="cuda"), old // p].long()
    kept = torch.zeros(n, dtype=torch.long, device="cuda").scatter(0, first_page, half)
    touched = torch.zeros(n, dtype=torch.bool, device="cuda").scatter(0, page, True)
    before = torch.frexp(scale)[1] - 1
    after = torch.where((kept > 0)[:, None], torch.maximum(want, before), want)
    after = torch.where(touched[:, None], after, before)
    view = codes.view(n, h, p // 8, d // 16, 8, 16).permute(0, 1, 2, 4, 3, 5) if key else codes.view(n, h, p // 16, d, 16).permute(0, 1, 2, 4, 3)
    block = view.reshape(n, h, p, d).view(torch.float8_e4m3fn)
    grown = (kept > 0)[:, None] & touched[:, None] & (after > before)
    lower = (block.float() * torch.exp2((before - after).float())[..., None, None]).to(torch.float8_e4m3fn)
    older = torch.arange(p, device="cuda")[None, None, :, None] < kept[:, None, None, None]
    block = torch.where(older & grown[..., None, None], lower.view(torch.uint8), block.view(torch.uint8))
    block[page, :, slot] = (rows * torch.exp2(-after[page].float())[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes.copy_(_key_layout(block) if key else _value_layout(block))
    scale.copy_(torch.exp2(after.float()))


def _gathered(s, codes, scale, key):
    """[sequences][heads][pages of the table * page][dim] in 32 bits."""
    c = s["case"]
    n, h, p, d = s["pages"], c["heads"], c["page"], c["dim"]
    at = s["table"].clamp(min=0).long()
    if key:
        x = codes.view(n, h, p // 8, d // 16, 8, 16)[at].permute(0, 2, 1, 3, 5, 4, 6)
    else:
        x = codes.view(n, h, p // 16, d, 16)[at].permute(0, 2, 1, 3, 5, 4)
    x = x.reshape(c["seqs"], h, at.shape[1], p, d).view(torch.float8_e4m3fn).float()
    return (x * scale[at].permute(0, 2, 1)[..., None, None]).reshape(c["seqs"], h, -1, d)


def _attention(s):
    c = s["case"]
    h, d, group, t = c["heads"], c["dim"], c["q_heads"] // c["heads"], DTYPES[c["dtype"]]
    k, v = _gathered(s, s["k"], s["k_scale"], True), _gathered(s, s["v"], s["v_scale"], False)
    new = (s["first"][1:] - s["first"][:-1])[:, None]
    i = torch.arange(s["max_new"], device="cuda")[None, :]
    row = (s["first"][:-1, None] + torch.minimum(i, new - 1)).long()
    q = s["q"].float()[row].view(c["seqs"], -1, h, group, d).permute(0, 2, 1, 3, 4).reshape(c["seqs"], h, -1, d)
    score = torch.matmul(q, k.transpose(-1, -2)) * d ** -0.5
    place = (s["len"][:, None] - new + i)[..., None]
    key = torch.arange(k.shape[2], device="cuda")[None, None, :]
    seen = key < s["len"][:, None, None]
    if c["causal"]:
        seen = seen & (key <= place)
    if c["window"]:
        seen = seen & (key > place - c["window"])
    score = score.view(c["seqs"], h, s["max_new"], group, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(c["seqs"], h, -1, score.shape[-1]), v).view(c["seqs"], h, s["max_new"], group, d)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log())[..., 0]
    r = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["first"][1:], r, right=True)
    at = (r - s["first"][b]).long()
    out = out[b, :, at].reshape(-1, c["q_heads"], d).to(t)
    return dict(out=out, lse=lse[b, :, at].reshape(-1, c["q_heads"])) if c["lse"] else out


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    if c["op"] == "rotary":
        return _rotated(state, state["x"], c["inverse"]).to(DTYPES[c["dtype"]])
    if c["op"] == "append":
        _appended_block(state, _rotated(state, state["new_k"]), state["k"], state["k_scale"], True)
        _appended_block(state, state["new_v"].float(), state["v"], state["v_scale"], False)
        return _appended(state, _rotated(state, state["q"]).to(DTYPES[c["dtype"]]))
    return _attention(state)


# ---- the definitions in 64 bits


def _turn(s, x, inverse=False):
    """The rotation as a product of complex numbers."""
    c, rot = s["case"], s["case"]["rot"]
    edges = [0]
    for n in s["sections"]:
        edges.append(edges[-1] + n)
    angle = torch.empty(x.shape[0], rot // 2, dtype=torch.float64, device="cuda")
    for a in range(c["axes"]):
        angle[:, edges[a] : edges[a + 1]] = s["pos"][a].double()[:, None] * s["freq"][edges[a] : edges[a + 1]].double()
    unit = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, None, :]
    y = x.double().clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["adjacent"] else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(y[..., first].clone(), y[..., second].clone()) * unit
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _nearest_code(x):
    """The e4m3 value nearest to x (|x| <= 448), ties to the even one, in 64 bits."""
    exponent = (torch.frexp(x.abs())[1] - 1).clamp(min=-6)
    step = torch.exp2(exponent.double() - 3)
    return torch.round(x / step) * step


def _exact_append(s, rows, codes, scale, key):
    c = s["case"]
    n, h, p, d = s["pages"], c["heads"], c["page"], c["dim"]
    values = codes.view(torch.float8_e4m3fn).double()
    values = values.view(n, h, p // 8, d // 16, 8, 16).permute(0, 1, 2, 4, 3, 5) if key else values.view(n, h, p // 16, d, 16).permute(0, 1, 2, 4, 3)
    values, scale = values.reshape(n, h, p, d).clone(), scale.double().clone()
    first, length, table = s["first"].tolist(), s["len"].tolist(), s["table"].tolist()
    for b in range(c["seqs"]):
        place = length[b] - (first[b + 1] - first[b])
        row = first[b]
        while row < first[b + 1]:
            slot = place % p
            take = min(p - slot, first[b + 1] - row)
            page, new = table[b][place // p], rows[row : row + take].transpose(0, 1)
            power = torch.ceil(torch.log2(new.abs().amax(dim=(1, 2)) / 448)).clamp(-40, 40)
            fit = torch.exp2(power)
            if slot:
                grown = torch.maximum(fit, scale[page])
                values[page, :, :slot] = torch.where((grown > scale[page])[:, None, None], _nearest_code(values[page, :, :slot] * (scale[page] / grown)[:, None, None]), values[page, :, :slot])
                fit = grown
            scale[page] = fit
            values[page, :, slot : slot + take] = _nearest_code(new / fit[:, None, None])
            row, place = row + take, place + take
    values = values.view(n, h, p // 8, 8, d // 16, 16).permute(0, 1, 2, 4, 3, 5) if key else values.view(n, h, p // 16, 16, d).permute(0, 1, 2, 4, 3)
    return values.reshape(-1), scale


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "rotary":
        return _turn(s, s["x"], c["inverse"])
    if c["op"] == "append":
        k, ks = _exact_append(s, _turn(s, s["new_k"]), s["k"], s["k_scale"], True)
        v, vs = _exact_append(s, s["new_v"].double(), s["v"], s["v_scale"], False)
        return dict(q=_turn(s, s["q"]), k=k, v=v, k_scale=ks, v_scale=vs)
    h, p, d, group = c["heads"], c["page"], c["dim"], c["q_heads"] // c["heads"]
    keys = s["k"].view(torch.float8_e4m3fn).view(-1, h, p // 8, d // 16, 8, 16)
    values = s["v"].view(torch.float8_e4m3fn).view(-1, h, p // 16, d, 16)
    first, length = s["first"].tolist(), s["len"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b in range(c["seqs"]):
        n, size = first[b + 1] - first[b], length[b]
        used = s["table"][b, : -(-size // p)].long()
        place = torch.arange(size - n, size, device="cuda")[:, None]
        at = torch.arange(size, device="cuda")[None, :]
        bias = torch.zeros(n, size, dtype=torch.float64, device="cuda")
        if c["causal"]:
            bias[at > place] = -math.inf
        if c["window"]:
            bias[at <= place - c["window"]] = -math.inf
        for head in range(h):
            k = (keys[used, head].double().permute(0, 1, 3, 2, 4).reshape(-1, p * d) * s["k_scale"][used, head].double()[:, None]).view(-1, d)[:size]
            v = (values[used, head].double().transpose(-1, -2).reshape(-1, p * d) * s["v_scale"][used, head].double()[:, None]).view(-1, d)[:size]
            for g in range(group):
                j = head * group + g
                logit = s["q"][first[b] : first[b + 1], j].double() @ k.T / math.sqrt(d) + bias
                total = torch.logsumexp(logit, dim=-1)
                lse[first[b] : first[b + 1], j] = total
                out[first[b] : first[b + 1], j] = torch.nan_to_num(torch.exp(logit - total[:, None])) @ v
    return dict(out=out, lse=lse) if c["lse"] else out
