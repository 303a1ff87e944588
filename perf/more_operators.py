"""The rest of an attention layer around the 8-bit paged cache, as timed cases.

Every case is one call that a serving process makes per layer:

* ``axes``    rotary positions with several axes: each token has a time, a
              height and a width, and each pair of a head's elements turns by one
              of them, in sections one after the other or in turn.  The queries of
              a batch, or its keys on their way into the cache (``append``).
* ``first``   attention over the cache with a sliding window and the sequence's
              first few tokens, which every query sees however far it is.
* ``shared``  attention of sequences that begin with the same prompt: its pages
              stand in every sequence's row of the block table, and the call says
              which sequences share how much.
* ``norm``    what stands between two blocks of a layer: the norm after one, its
              gate and scale, the sum with the residual stream, the norm before
              the next, whose result may go out as e4m3 codes with one scale for
              128 elements, as an FP8 linear layer reads it.

With ``own`` the package's entry points are called; without it the same is
computed with elementary torch operations in 32 bits.

The cache: codes [pages, kv heads, page, D] and scales [pages, kv heads,
page / block]; ``pages`` [B, n] lists the pages of a sequence in order.
"""

import math
import os
import random
import sys

import torch

own = False

BF16, F16, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
DTYPES = {"bf16": BF16, "f16": F16, "f32": F32}


def listed():
    return [
        # the queries of a decode step of 16 sequences: latency alone
        dict(name="axes_t16", kind="axes", T=16, H=32, D=128, rot=128, sections="16,24,24",
             spread=False, layout="half", dtype="bf16", context=32768),
        # all queries of a large prefill of pictures, the axes in turn
        dict(name="axes_t16384", kind="axes", T=16384, H=32, D=128, rot=128, sections="24,20,20",
             spread=True, layout="half", dtype="bf16", context=32768),
        # the keys and values of prompts of odd lengths behind what the cache has
        dict(name="append_b5_t4099", kind="append", B=5, T=4099, Hkv=8, D=128, page=64, block=64,
             rot=128, sections="16,24,24", spread=False, layout="half", dtype="bf16", context=2048),
        # one sequence answers at the end of a long conversation
        dict(name="first_b1_c20000_w1024", kind="first", B=1, T=1, Hq=32, Hkv=8, D=128, page=64,
             block=64, context=20000, window=1024, first=4, sink=False, dtype="bf16"),
        # a large decode batch of mixed lengths, a longer window and a sink
        dict(name="first_b128_c30000_w4096", kind="first", B=128, T=128, Hq=64, Hkv=8, D=128, page=64,
             block=64, context=30000, window=4096, first=128, sink=True, dtype="bf16"),
        # prompt chunks of odd lengths behind cached prefixes, small heads
        dict(name="first_b4_t5001_w1000", kind="first", B=4, T=5001, Hq=64, Hkv=8, D=64, page=16,
             block=16, context=12000, window=1000, first=20, sink=False, dtype="f16"),
        # a few samples of one short prompt
        dict(name="shared_b4_p1500", kind="shared", B=4, T=4, groups=1, Hq=32, Hkv=8, D=128, page=64,
             block=64, prefix=1500, rest=200, sink=False, dtype="bf16"),
        # chats under one system prompt, two draft tokens each
        dict(name="shared_b60_p8192_q2", kind="shared", B=60, T=120, groups=1, Hq=32, Hkv=8, D=128,
             page=64, block=32, prefix=8192, rest=1500, sink=False, dtype="bf16"),
        # a large batch of questions on two long documents
        dict(name="shared_b128_p32768_g2", kind="shared", B=128, T=128, groups=2, Hq=64, Hkv=4, D=128,
             page=64, block=64, prefix=32768, rest=3000, sink=True, dtype="bf16"),
        # a decode step of 8 sequences: the sum and the norm before an FP8 layer
        dict(name="norm_t8_h4096", kind="norm", T=8, H=4096, after=False, gate="none", scale=1.0,
             dtype="bf16", res="bf16", quant=True),
        # chunks of prompts: a norm on either side, a gate for each element, a residual stream in fp32
        dict(name="norm_t1900_h7168", kind="norm", T=1900, H=7168, after=True, gate="rows", scale=0.7,
             dtype="bf16", res="f32", quant=False),
        # a large prefill: a norm on either side, a gate for each channel, codes for an FP8 layer
        dict(name="norm_t16384_h4096", kind="norm", T=16384, H=4096, after=True, gate="vector", scale=0.5,
             dtype="bf16", res="bf16", quant=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _sections(rng, pairs):
    """Pairs of each axis: two or three of them, of any sizes."""
    if rng.random() < 0.3:
        n = rng.randint(1, pairs - 1)
        return "%d,%d" % (n, pairs - n)
    a = rng.randint(1, pairs - 2)
    b = rng.randint(1, pairs - a - 1)
    return "%d,%d,%d" % (a, b, pairs - a - b)


def draw(rng):
    kind = rng.choice(["axes", "append", "first", "first", "shared", "shared", "norm", "norm"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "norm":
        H = rng.choice([512, 1000, 1536, 2048, 4096, 4100, 5120, 7168])
        res = rng.choice([dtype, dtype, "f32"])
        after = rng.random() < 0.5
        gate = rng.choice(["none", "vector", "rows"])
        quant = H % 128 == 0 and rng.random() < 0.5
        T = _log(rng, 1, min(16384, 16384 * 4096 // (H * (1 + (res == "f32") + (gate == "rows")))))
        return dict(kind=kind, T=T, H=H, after=after, gate=gate, scale=rng.choice([1.0, 0.5, 1.7]),
                    dtype=dtype, res=res, quant=quant)
    if kind == "axes":
        D = rng.choice([64, 80, 128, 128, 256])
        H = rng.choice([1, 7, 16, 32, 64])
        rot = rng.choice([D, D, D // 2])
        dtype = rng.choice([dtype, "f32"])
        most = 16384 * 32 * 128 * 2 // (H * D * (4 if dtype == "f32" else 2))
        return dict(kind=kind, T=_log(rng, 1, min(16384, most)), H=H, D=D, rot=rot,
                    sections=_sections(rng, rot // 2), spread=rng.random() < 0.5,
                    layout=rng.choice(["half", "half", "interleaved"]), dtype=dtype,
                    context=rng.choice([4096, 32768]))
    D, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64) if b <= page])
    Hkv = rng.choice([1, 2, 4, 8])
    if kind == "append":
        B = _log(rng, 1, 256)
        T = B if rng.random() < 0.4 else _log(rng, B, min(8192, 8192 * 1024 // (Hkv * D)))
        rot = rng.choice([D, D, D // 2])
        return dict(kind=kind, B=B, T=T, Hkv=Hkv, D=D, page=page, block=block, rot=rot,
                    sections=_sections(rng, rot // 2), spread=rng.random() < 0.5,
                    layout=rng.choice(["half", "half", "interleaved"]), dtype=dtype,
                    context=_log(rng, 1, 8192))
    Hq = Hkv * rng.choice([1, 4, 8, 16] if Hkv < 8 else [1, 4, 8])
    extra = dict(Hq=Hq, Hkv=Hkv, D=D, page=page, block=block, sink=rng.random() < 0.3, dtype=dtype)
    if kind == "shared":
        B = _log(rng, 2, 128)
        each = rng.choice([1, 1, 1, 2, 4, 33])
        each = max(1, min(each, 128 * 64 * 128 // (B * Hq * D)))
        room = 128 * 35768 * 512 // (B * Hkv * D)
        prefix = _log(rng, 64, min(32768, room // 2))
        prefix = min(prefix, 128 * 64 * 128 * 24000 // (B * each * Hq * D))
        return dict(kind=kind, B=B, T=B * each, groups=rng.choice([1, 1, min(2, B), min(3, B)]),
                    prefix=prefix, rest=each + _log(rng, 1, min(4000, room // 4)), **extra)
    window, first = _log(rng, 100, 5000), rng.choice([1, 4, 16, 64, 100, 300])
    extra.update(window=window, first=first)
    if rng.random() < 0.6:  # decode, or a few draft tokens
        B = _log(rng, 1, 128)
        context = _log(rng, 100, min(60000, 30000 * 128 * 1024 // (B * Hkv * D)))
        return dict(kind=kind, B=B, T=B * rng.choice([1, 1, 1, 2, 4]), context=context, **extra)
    B = rng.choice([1, 1, 2, 5])
    T = _log(rng, 64, 6000)
    T = max(4 * B + 1, min(T, T * 4096 // (Hq * D) if Hq * D > 4096 else T))
    context = T + _log(rng, 1, 12000)
    context = max(T + 1, min(context, 12000 * 5001 * 4096 // (2 * T * Hq * D)))
    return dict(kind=kind, B=B, T=T, context=context, **extra)


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _frequencies(c):
    """Radians per position of each pair, in 64 bits."""
    return 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])


def _table(c):
    """cos and sin [positions, pairs, 2] in fp32, from angles in 64 bits."""
    at = torch.arange(c["context"] + c["T"], dtype=torch.float64, device="cuda")
    angle = at[:, None] * _frequencies(c)[None, :]
    return torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1).float()


def _axis_of_pair(c):
    """The axis that each pair turns by: sections one after the other, or (``spread``) the axes
    in turn, as long as one has pairs left."""
    sizes = [int(n) for n in c["sections"].split(",")]
    if not c["spread"]:
        return [a for a, n in enumerate(sizes) for _ in range(n)]
    return [a for turn in range(max(sizes)) for a, n in enumerate(sizes) if turn < n]


def _axis_positions(c, g, T):
    """int32 [axes, T]: text (the same position on all axes) between pictures of 8 to 32 patches a
    side, whose height and width count on from the time of their first patch."""
    axes = c["sections"].count(",") + 1
    time = torch.randint(0, c["context"], (T,), generator=g, device="cuda")
    grid = torch.randint(0, 32, (axes, T), generator=g, device="cuda")
    grid[0] = 0
    picture = torch.rand(T, generator=g, device="cuda") < 0.7
    return (time + torch.where(picture, grid, 0)).clamp_max(c["context"] + T - 1).to(torch.int32).contiguous()


def _lengths(c):
    """Per sequence: its tokens in this call, and its tokens when the call is over (attention) or
    before it (`append`).  The batch's sum is the case's; which sequence has which is the seed's."""
    B, T = c["B"], c["T"]
    if c["kind"] == "shared":  # behind the prefix, here
        each = T // B
        return [each] * B, [each + (c["rest"] - each) * (i + 1) // B for i in range(B)]
    if T % B == 0 and T // B <= 4:
        new = [T // B] * B
    else:  # one token for a third of the sequences, the others in growing chunks
        share = [max(0, i - B // 3 + 1) for i in range(B)]
        new = [1 + (T - B) * s // sum(share) for s in share]
        new[-1] += T - sum(new)
    if c["kind"] == "append":
        have = [int(c["context"] * i / max(1, B - 1)) if B > 1 else c["context"] for i in range(B)]
    else:
        spread = [(i + 1.0) / B for i in range(B)]
        have = [max(n, int(round(c["context"] * s))) for n, s in zip(new, spread)]
        have[-1] = max(have[-1], c["context"])
    return new, have


def _groups(c):
    """`shared`: first sequence of each group and the end, and the groups' prefixes, growing."""
    n, B = c["groups"], c["B"]
    return [B * i // n for i in range(n + 1)], [max(1, c["prefix"] * (i + 1) // n) for i in range(n)]


def _batch(c, seed):
    new, have = _lengths(c)
    r = random.Random(seed)
    both = list(zip(new, have))
    r.shuffle(both)
    return [b[0] for b in both], [b[1] for b in both], r


def _pages(counts, r, group=None, common=None):
    """Page ids in the order of an allocator that has run for a while; -1 behind a sequence's last.
    group: each sequence's; common: how many of its first pages are those of all of the group."""
    group, common = group or list(range(len(counts))), common or [0] * len(counts)
    total = sum(common) + sum(n - common[g] for n, g in zip(counts, group))
    ids = list(range(total))
    r.shuffle(ids)
    begin = [[ids.pop() for _ in range(n)] for n in common]
    rows, width = [], max(counts)
    for n, g in zip(counts, group):
        rows.append(begin[g] + [ids.pop() for _ in range(n - common[g])] + [-1] * (width - n))
    return _int32(rows), total


def _codes(g, pages, H, page, D, block):
    """Codes and power-of-two scales of normally distributed rows whose size differs from block to block."""
    nb = page // block
    e = torch.randint(-9, -5, (pages, H, nb), generator=g, device="cuda")
    codes = torch.empty(pages, H, page, D, dtype=FP8, device="cuda")
    flat = codes.view(torch.uint8).view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = _randn(g, n).mul_(80.0).clamp_(-448.0, 448.0).to(FP8).view(torch.uint8)
    return codes, torch.exp2(e.float())


def _inputs(c, seed):
    """The case's tensors, from the seed alone."""
    g = _gen(seed)
    if c["kind"] == "axes":
        x = _randn(g, c["T"], c["H"], c["D"]).to(DTYPES[c["dtype"]])
        return dict(x=x, positions=_axis_positions(c, g, c["T"]), table=_table(c),
                    axes=torch.tensor(_axis_of_pair(c), device="cuda"))
    if c["kind"] == "norm":
        T, H, dt = c["T"], c["H"], DTYPES[c["dtype"]]
        size = torch.exp2(_randn(g, T, 1))
        t = dict(x=(_randn(g, T, H) * size).to(dt), residual=(_randn(g, T, H) * 3.0).to(DTYPES[c["res"]]))
        t["before"] = 1.0 + 0.2 * _randn(g, H)
        t["after"] = 1.0 + 0.2 * _randn(g, H) if c["after"] else None
        t["gate"] = None
        if c["gate"] != "none":
            t["gate"] = torch.tanh(_randn(g, *((T, H) if c["gate"] == "rows" else (H,)))).to(dt)
        return t
    new, have, r = _batch(c, seed)
    page, block, D, H = c["page"], c["block"], c["D"], c["Hkv"]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    group = common = None
    t = dict(cu=_int32(cu))
    if c["kind"] == "shared":
        edge, prefix = _groups(c)
        group = [i for i in range(c["groups"]) for _ in range(edge[i + 1] - edge[i])]
        common = [p // page for p in prefix]
        have = [prefix[j] + h for j, h in zip(group, have)]
        t.update(cu_groups=_int32(edge), shared=_int32(prefix))
    t.update(have=_int32(have), most=max(new), longest=max(have))
    if c["kind"] == "append":
        t["pages"], total = _pages([-(-(n + h) // page) for n, h in zip(new, have)], r)
        t["k"], t["v"] = _new_rows(c, g)
        (t["kc"], t["ks"]), (t["vc"], t["vs"]) = [_codes(g, total, H, page, D, block) for _ in range(2)]
        t.update(table=_table(c), positions=_axis_positions(c, g, c["T"]),
                 axes=torch.tensor(_axis_of_pair(c), device="cuda"))
        return t
    t["pages"], total = _pages([-(-h // page) for h in have], r, group, common)
    (t["kc"], t["ks"]), (t["vc"], t["vs"]) = [_codes(g, total, H, page, D, block) for _ in range(2)]
    for b, h in enumerate(have):  # what lies behind a sequence's last token was never written
        if h % page:
            last = int(t["pages"][b, h // page])
            for code, scale in ((t["kc"], t["ks"]), (t["vc"], t["vs"])):
                code.view(torch.uint8)[last, :, h % page:] = 0x7F
                scale[last, :, -(-(h % page) // block):] = float("nan")
    t["q"] = _randn(g, c["T"], c["Hq"], D).to(DTYPES[c["dtype"]])
    t["sink"] = _randn(g, c["Hq"]) if c["sink"] else None
    return t


def _new_rows(c, g):
    """New keys and values, as views of a fused projection's rows, of sizes that differ from token to token."""
    T, H, D = c["T"], c["Hkv"], c["D"]
    rows = _randn(g, T, 2 * H, D) * torch.exp2(_randn(g, T, 1, 1))
    rows = rows.to(DTYPES[c["dtype"]])
    return rows[:, :H], rows[:, H:]


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if "axes" in s:  # which axis a pair turns by: a model's own, made once
        s["axes8"] = s["axes"].to(torch.uint8)
    if "B" in case and case["T"] == case["B"]:
        s["cu"] = None  # one token each: the lengths of the chunks go without saying
    return s


# ------------------------------------------------------------- plain forms


def _rotate(x, table, positions, axes, layout):
    """fp32 [T, H, D] with the first pairs rotated, each by its axis' position of the token."""
    pair = torch.arange(axes.numel(), device="cuda")
    cos, sin = table[positions.long()[axes].t(), pair][:, None].unbind(-1)  # [T, 1, pairs]
    rot = 2 * pair.numel()
    y = x.float().clone()
    part = y[..., :rot]
    if layout == "half":
        a, b = part[..., :rot // 2], part[..., rot // 2:]
    else:
        a, b = part[..., 0::2], part[..., 1::2]
    p, q = a * cos - b * sin, b * cos + a * sin
    if layout == "half":
        part[..., :rot // 2], part[..., rot // 2:] = p, q
    else:
        part[..., 0::2], part[..., 1::2] = p, q
    return y


def _token_places(s):
    """Per new token: its sequence and its position there."""
    c = s["case"]
    row = torch.arange(c["T"], device="cuda")
    if s["cu"] is None:
        seq, at = row, torch.zeros_like(row)
    else:
        seq = torch.bucketize(row, s["cu"][1:].long(), right=True)
        at = row - s["cu"].long()[seq]
    return seq, s["have"].long()[seq] + at


def _scale_of(amax):
    """The smallest power of two, 2^-100 at least, that brings amax down to 448."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -100).clamp_min(-100))


def _append_one(s, x, codes, scales, seq, at):
    """Values x fp32 [T, H, D] into codes and scales, both in place."""
    c = s["case"]
    page, block = c["page"], c["block"]
    nb, H, D = page // block, c["Hkv"], c["D"]
    to_page = s["pages"].long()[seq, at // page]
    spot = at % page
    piece = to_page * nb + spot // block  # the block of tokens that a token is in
    amax = torch.zeros(codes.shape[0] * nb, H, device="cuda")
    amax.scatter_reduce_(0, piece[:, None].expand(-1, H), x.abs().amax(-1), "amax")
    fresh = _scale_of(amax).view(-1, nb, H).transpose(1, 2)
    # blocks that hold a sequence's earlier tokens
    have = s["have"].long()
    room = torch.arange(have.numel(), device="cuda")
    old_page = s["pages"].long()[room, have // page]
    old_piece = have % page // block
    begun = (have % block > 0)[:, None]
    was = scales[old_page, :, old_piece]
    now = torch.where(begun, torch.maximum(was, fresh[old_page, :, old_piece]), fresh[old_page, :, old_piece])
    slot = (old_piece * block)[:, None] + torch.arange(block, device="cuda")
    kept = codes.view(torch.uint8)[old_page[:, None], :, slot].view(FP8).float()  # [B, block, H, D]
    again = (kept * was[:, None, :, None] / now[:, None, :, None]).to(FP8)
    mine = (slot < (have % page)[:, None])[:, :, None, None] & begun[:, :, None, None]
    bytes_ = torch.where(mine, again.view(torch.uint8), kept.to(FP8).view(torch.uint8))
    codes.view(torch.uint8)[old_page[:, None], :, slot] = bytes_
    scale = fresh.clone()
    scale[old_page, :, old_piece] = now
    wrote = torch.zeros(codes.shape[0] * nb, dtype=torch.bool, device="cuda")
    wrote[piece] = True
    scales.copy_(torch.where(wrote.view(-1, 1, nb), scale, scales))
    mult = scales[to_page, :, spot // block]
    codes.view(torch.uint8)[to_page, :, spot] = (x / mult[:, :, None]).to(FP8).view(torch.uint8)


def _plain_append(s):
    seq, at = _token_places(s)
    k = _rotate(s["k"], s["table"], s["positions"], s["axes"], s["case"]["layout"])
    _append_one(s, k, s["kc"], s["ks"], seq, at)
    _append_one(s, s["v"].float(), s["vc"], s["vs"], seq, at)
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _plain_attn(s):
    c = s["case"]
    B, Hq, Hkv, D, page, block = c["B"], c["Hq"], c["Hkv"], c["D"], c["page"], c["block"]
    L, n, G = s["longest"], s["most"], Hq // Hkv
    key = torch.arange(L, device="cuda")
    have = s["have"].long()
    there = key < have[:, None]  # [B, L]
    at = s["pages"].long()[:, key // page].clamp_min(0)
    spot = (key % page).expand(B, L)

    def rows(codes, scales):
        x = codes.view(torch.uint8)[at, :, spot].view(FP8).float() * scales[at, :, spot // block][..., None]
        return torch.where(there[..., None, None], x, 0.0).permute(0, 2, 1, 3).contiguous()  # [B, Hkv, L, D]

    first = torch.arange(B, device="cuda") if s["cu"] is None else s["cu"][:-1].long()
    count = torch.ones_like(first) if s["cu"] is None else s["cu"].long().diff()
    i = torch.arange(n, device="cuda")
    pick = torch.where(i < count[:, None], first[:, None] + i, 0)
    q = s["q"].float()[pick].view(B, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B * Hkv, n * G, D)
    k = rows(s["kc"], s["ks"]).view(B * Hkv, L, D)
    score = torch.bmm(q, k.transpose(1, 2).contiguous()).view(B, Hkv, n, G, L) * D ** -0.5
    del k
    place = have[:, None] - count[:, None] + i  # [B, n], the queries' own positions
    seen = (key <= place[..., None]) & there[:, None]
    if c["kind"] == "first":
        seen &= (key > place[..., None] - c["window"]) | (key < c["first"])
    score.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].view(1, Hkv, 1, G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top > float("-inf"), top, 0.0)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(sink - top)
    v = rows(s["vc"], s["vs"]).view(B * Hkv, L, D)
    o = torch.bmm(p.view(B * Hkv, n * G, L), v).view(B, Hkv, n, G, D)
    o = torch.where(total > 0, o / total, 0.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(B, n, Hq, D)
    return o[i < count[:, None]].to(DTYPES[c["dtype"]])


EPS = 1e-6


def _plain_norm(s):
    c = s["case"]

    def norm(x, weight):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight

    u = s["x"].float()
    if s["after"] is not None:
        u = norm(u, s["after"])
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = s["residual"].float() + c["scale"] * u
    y = norm(h, s["before"])
    h = h.to(s["residual"].dtype)
    if not c["quant"]:
        return h, y.to(s["x"].dtype)
    parts = y.view(c["T"], -1, 128)
    scale = parts.abs().amax(-1).clamp_min(1e-4) / 448.0
    return h, (parts * (1.0 / scale)[..., None]).to(FP8).view_as(y), scale


def run(s):
    c = s["case"]
    if own:
        return _run_own(s)
    if c["kind"] == "axes":
        return _rotate(s["x"], s["table"], s["positions"], s["axes"], c["layout"]).to(DTYPES[c["dtype"]])
    if c["kind"] == "append":
        return _plain_append(s)
    return _plain_norm(s) if c["kind"] == "norm" else _plain_attn(s)


_modules = []


def _run_own(s):
    c = s["case"]
    if not _modules:
        _package()
    R, P, N = _modules
    if c["kind"] == "axes":
        return R.rotary(s["x"], s["table"], s["positions"], axes=s["axes8"],
                        interleaved=c["layout"] == "interleaved")
    if c["kind"] == "norm":
        h, y = N.residual_norm(s["x"], s["residual"], s["before"], after=s["after"], gate=s["gate"],
                               scale=c["scale"], eps=EPS, quant=c["quant"])
        return (h, *y) if c["quant"] else (h, y)
    cache = P.PagedKV(s["kc"], s["vc"], s["ks"], s["vs"])
    if c["kind"] == "append":
        P.append_kv(cache, s["k"], s["v"], s["pages"], s["have"], cu_tokens=s["cu"], table=s["table"],
                    positions=s["positions"], axes=s["axes8"], interleaved=c["layout"] == "interleaved")
        return cache.k, cache.v, cache.k_scale, cache.v_scale
    if c["kind"] == "first":
        return P.paged_attn(s["q"], cache, s["pages"], s["have"], cu_tokens=s["cu"], window=c["window"],
                            first=c["first"], sink=s["sink"])
    return P.paged_attn(s["q"], cache, s["pages"], s["have"], cu_tokens=s["cu"], sink=s["sink"],
                        cu_groups=s["cu_groups"], shared=s["shared"])


def _package():
    """The package's modules, imported by the first call with `own`."""
    at = os.path.join(os.getcwd(), "sglang-lite_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from sglang_lite_amd import norms, paged_kv, rotary

    _modules[:] = [rotary, paged_kv, norms]


# -------------------------------------------------------------------- work


def work(case):
    c = case
    if c["kind"] == "axes":
        n = c["T"] * c["H"] * c["D"]
        size = 4 if c["dtype"] == "f32" else 2
        axes = c["sections"].count(",") + 1
        return dict(bytes=2 * n * size + c["T"] * (4 * axes + 4 * c["rot"]), flops=3 * c["T"] * c["H"] * c["rot"])
    if c["kind"] == "norm":
        T, H, res = c["T"], c["H"], 4 if c["res"] == "f32" else 2
        gate = dict(none=0, vector=2 * H, rows=2 * T * H)[c["gate"]]
        y = T * H + T * H // 32 if c["quant"] else 2 * T * H
        return dict(bytes=2 * T * H + 2 * res * T * H + gate + y + 4 * H * (1 + c["after"]),
                    flops=T * H * (6 + 4 * c["after"] + (c["gate"] != "none") + 2 * c["quant"]))
    new, have = _lengths(c)
    H, D = c["Hkv"], c["D"]
    if c["kind"] == "append":
        n, axes = c["T"] * H * D, c["sections"].count(",") + 1
        return dict(bytes=2 * n * 3 + c["T"] * (4 * c["rot"] + 4 * axes), flops=3 * c["T"] * H * c["rot"] + 4 * n)
    read = pairs = 0
    if c["kind"] == "shared":
        edge, prefix = _groups(c)
        read = sum(prefix) + sum(have)
        pairs = sum(c["T"] // c["B"] * (b - a) * p for a, b, p in zip(edge, edge[1:], prefix))
        pairs += sum(n * (h - n) + n * (n + 1) // 2 for n, h in zip(new, have))
    else:
        for n, h in zip(new, have):
            w, f = c["window"], c["first"]
            low = max(0, h - n - w + 1)  # where the window of its first query begins
            read += h - low + min(f, low)
            for p in range(h - n, h):
                pairs += min(p + 1, w) + min(f, max(0, p + 1 - w))
    row = 2 * H * (D + 4 / c["block"])
    return dict(bytes=read * row + 4 * c["T"] * c["Hq"] * D, flops=4 * pairs * c["Hq"] * D)


# ------------------------------------------------------------------- exact


def _exact_rotated(c, x, positions):
    """Rotation as a product of complex numbers, angles from the definition."""
    at = torch.stack([positions[a] for a in _axis_of_pair(c)], dim=1).double()  # [T, pairs]
    turn = torch.polar(torch.ones_like(at), at * _frequencies(c))[:, None]
    x = x.double()
    rot = c["rot"]
    part, tail = x[..., :rot], x[..., rot:]
    if c["layout"] == "half":
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * turn
        part = torch.cat([z.real, z.imag], dim=-1)
    else:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * turn
        part = torch.view_as_real(z).reshape(part.shape)
    return torch.cat([part, tail], dim=-1)


def _exact_append(c, t):
    """Sequence by sequence and block by block; codes before their rounding, as the values are then."""
    new, have = t["cu"].diff().tolist(), t["have"].tolist()
    page, block = c["page"], c["block"]
    pages = t["pages"].tolist()
    out = []
    for x, codes, scales in ((_exact_rotated(c, t["k"], t["positions"]), t["kc"], t["ks"]),
                             (t["v"].double(), t["vc"], t["vs"])):
        # the scale goes by the largest value as it is in 32 bits, the type it is found in
        codes, scales, row = codes.double(), scales.double(), 0
        for b, (n, h) in enumerate(zip(new, have)):
            end, at = h + n, h
            while at < end:
                upto = min(end, (at // block + 1) * block)
                p, lo, hi = pages[b][at // page], at % page, (upto - 1) % page + 1
                piece, rows = lo // block, x[row:row + upto - at].transpose(0, 1)
                peak = rows.abs().amax((1, 2)).float().double()
                s = torch.exp2(torch.ceil(torch.log2(peak.clamp_min(2.0 ** -120) / 448.0)).clamp_min(-100))
                begin = piece * block
                if lo > begin:
                    s = torch.maximum(s, scales[p, :, piece])
                    codes[p, :, begin:lo] *= (scales[p, :, piece] / s)[:, None, None]
                codes[p, :, lo:hi] = rows / s[:, None, None]
                scales[p, :, piece] = s
                row, at = row + upto - at, upto
        out.append((codes, scales))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _exact_attn(c, t):
    new, have = t["cu"].diff().tolist(), t["have"].tolist()
    page, block, D, G = c["page"], c["block"], c["D"], c["Hq"] // c["Hkv"]
    o = torch.zeros(c["T"], c["Hq"], D, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, h) in enumerate(zip(new, have)):
        ids = t["pages"][b, :-(-h // page)].long()
        for j in range(c["Hkv"]):
            k, v = [(x[ids, j].double() * y[ids, j].double().repeat_interleave(block, 1)[..., None]).view(-1, D)[:h]
                    for x, y in ((t["kc"], t["ks"]), (t["vc"], t["vs"]))]
            kt = k.t().contiguous()
            for i0 in range(0, n, 512):
                i1 = min(n, i0 + 512)
                q = t["q"][row + i0:row + i1, j * G:(j + 1) * G].double().reshape(-1, D)
                at = torch.arange(h - n + i0, h - n + i1, device="cuda").repeat_interleave(G)
                spot = torch.arange(h, device="cuda")
                gap = at[:, None] - spot
                ok = gap >= 0
                if c["kind"] == "first":
                    ok &= (gap < c["window"]) | (spot < c["first"])
                e = torch.where(ok, (q @ kt) * D ** -0.5, float("-inf"))
                m = e.max(-1, keepdim=True).values.clamp_min(-1e300)
                w = torch.exp(e - m)
                den = w.sum(-1, keepdim=True)
                if t["sink"] is not None:
                    den = den + torch.exp(t["sink"][j * G:(j + 1) * G].double().repeat(i1 - i0)[:, None] - m)
                o[row + i0:row + i1, j * G:(j + 1) * G] = ((w @ v) / den).view(i1 - i0, G, D)
        row += n
    return o


def _exact_norm(c, t):
    x = t["x"].double()
    if t["after"] is not None:
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["H"] + EPS) * t["after"].double()
    if t["gate"] is not None:
        x = x * t["gate"].double()
    h = c["scale"] * x + t["residual"].double()
    y = h / torch.sqrt((h ** 2).sum(-1, keepdim=True) / c["H"] + EPS) * t["before"].double()
    if not c["quant"]:
        return h, y
    s = (y.reshape(-1, 128).abs().max(-1).values.clamp_min(1e-4) / 448.0).view(c["T"], -1)
    return h, y / s.repeat_interleave(128, 1), s  # (codes before their rounding)


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    if c["kind"] == "axes":
        return _exact_rotated(c, t["x"], t["positions"])
    if c["kind"] == "append":
        return _exact_append(c, t)
    return _exact_norm(c, t) if c["kind"] == "norm" else _exact_attn(c, t)
