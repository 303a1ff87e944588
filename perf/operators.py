"""Rotary positions, the 8-bit paged KV cache and the attention over it, as timed cases.

Every case is one call that a serving process makes per layer:

* ``rotary``  the positions of a batch's queries turned into rotations of pairs
              of elements: the whole head or a part of it, interleaved pairs or
              halves, forwards or back, tables scaled for long contexts or not.
* ``append``  new keys and values of a batch of sequences written to a paged
              cache of e4m3 codes with one power-of-two scale for each block of
              tokens and head, the keys rotated on the way.  A block that was
              begun before keeps its tokens: they are written again where the
              new ones need a larger scale.
* ``attn``    causal attention of the new queries of a batch over that cache, a
              window and an attention sink optional: one token a sequence
              (decode) or chunks of prompts (prefill).

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
        dict(name="rotary_t16", kind="rotary", T=16, H=32, D=128, rot=128, offset=0, layout="half",
             dtype="bf16", inverse=False, scaling="none", context=32768),
        # the latent heads of a prompt chunk: 64 of 512 elements, interleaved, a
        # long-context table, rotated back as the attention's outputs are
        dict(name="rotary_latent_t1900", kind="rotary", T=1900, H=64, D=512, rot=64, offset=448,
             layout="interleaved", dtype="bf16", inverse=True, scaling="yarn", context=131072),
        # all queries of a large prefill
        dict(name="rotary_t16384", kind="rotary", T=16384, H=32, D=128, rot=128, offset=0,
             layout="half", dtype="bf16", inverse=False, scaling="none", context=32768),
        # one new token for each of 64 sequences
        dict(name="append_b64", kind="append", B=64, T=64, Hkv=8, D=128, page=64, block=64,
             rot=128, layout="half", dtype="bf16", context=8192),
        # a step that mixes decode and prompt chunks of odd lengths, half of the head rotated
        dict(name="append_b24_t2301", kind="append", B=24, T=2301, Hkv=4, D=128, page=32, block=16,
             rot=64, layout="interleaved", dtype="f16", context=4096),
        # the prompts of a large prefill
        dict(name="append_b5_t16384", kind="append", B=5, T=16384, Hkv=8, D=128, page=64, block=64,
             rot=128, layout="half", dtype="bf16", context=2048),
        # one sequence begins to answer: the smallest call
        dict(name="attn_b1_c500", kind="attn", B=1, T=1, Hq=32, Hkv=8, D=128, page=64, block=64,
             context=500, window=0, sink=False, dtype="bf16"),
        # a decode step of 32 sequences of mixed lengths, four draft tokens each
        dict(name="attn_b32_c6000_q4", kind="attn", B=32, T=128, Hq=32, Hkv=8, D=128, page=64,
             block=32, context=6000, window=0, sink=False, dtype="bf16"),
        # few sequences with long contexts
        dict(name="attn_b3_c131072", kind="attn", B=3, T=3, Hq=64, Hkv=8, D=128, page=64, block=64,
             context=131072, window=0, sink=False, dtype="bf16"),
        # a large decode batch, one key head for sixteen query heads and a sink
        dict(name="attn_b128_c16384", kind="attn", B=128, T=128, Hq=64, Hkv=4, D=128, page=64,
             block=64, context=16384, window=0, sink=True, dtype="bf16"),
        # prompt chunks of odd lengths behind cached prefixes, small heads, window and sink
        dict(name="attn_b4_t2600_w1024", kind="attn", B=4, T=2600, Hq=64, Hkv=8, D=64, page=16,
             block=16, context=9000, window=1024, sink=True, dtype="f16"),
        # a whole prompt
        dict(name="attn_b1_t8192", kind="attn", B=1, T=8192, Hq=32, Hkv=8, D=128, page=64, block=64,
             context=8192, window=0, sink=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attn", "attn"])
    if kind == "rotary":
        D = rng.choice([64, 96, 128, 128, 256, 512])
        H = rng.choice([1, 7, 8, 16, 32, 64])
        rot = rng.choice([D, D // 2, 32])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        most = 16384 * 32 * 128 * 2 // (H * D * (4 if dtype == "f32" else 2))
        return dict(kind=kind, T=_log(rng, 1, min(16384, most)), H=H, D=D, rot=rot,
                    offset=rng.choice([0, D - rot]), layout=rng.choice(["half", "interleaved"]),
                    dtype=dtype, inverse=rng.random() < 0.3,
                    scaling=rng.choice(["none", "linear", "yarn"]),
                    context=rng.choice([4096, 32768, 131072]))
    D, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64) if b <= page])
    Hkv = rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        B = _log(rng, 1, 256)
        T = B if rng.random() < 0.4 else _log(rng, B, min(16384, 16384 * 1024 // (Hkv * D)))
        rot = rng.choice([D, D, D // 2, 0])
        return dict(kind=kind, B=B, T=T, Hkv=Hkv, D=D, page=page, block=block, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), dtype=dtype,
                    context=_log(rng, 1, 8192))
    Hq = Hkv * rng.choice([1, 4, 8, 16] if Hkv < 8 else [1, 4, 8])
    extra = dict(Hq=Hq, Hkv=Hkv, D=D, page=page, block=block, sink=rng.random() < 0.3, dtype=dtype,
                 window=rng.choice([0, 0, 0, 128, 1000]))
    if rng.random() < 0.6:  # decode, or a few draft tokens
        B = _log(rng, 1, 128)
        context = _log(rng, 16, min(131072, 16000 * 128 * 512 // (B * Hkv * D)))
        return dict(kind=kind, B=B, T=B * rng.choice([1, 1, 1, 2, 4]), context=context, **extra)
    B = rng.choice([1, 1, 2, 5])
    T = _log(rng, 64, 8192)
    T = max(4 * B + 1, min(T, T * 4096 // (Hq * D) if Hq * D > 4096 else T))
    context = T + _log(rng, 1, 16384)
    context = max(T + 1, min(context, 7600 * 8192 * 4096 // (2 * T * Hq * D)))
    return dict(kind=kind, B=B, T=T, context=context, **extra)


# ------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _frequencies(c, dtype=torch.float64):
    """Radians per position of each pair, and the factor of the rotated elements' length."""
    rot, base = c["rot"], 10000.0
    freq = base ** (-torch.arange(0, rot, 2, dtype=dtype, device="cuda") / rot)
    scaling = c.get("scaling", "none")
    if scaling == "linear":
        return freq / 8.0, 1.0
    if scaling == "yarn":  # 4096 positions stretched to `context`: slow pairs by the factor, fast ones not
        factor, original = c["context"] / 4096.0 if c["context"] > 4096 else 2.0, 4096

        def pair(turns):
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=dtype, device="cuda") - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _table(c):
    """cos and sin [positions, pairs, 2] in fp32, from angles in 64 bits."""
    freq, length = _frequencies(c)
    at = torch.arange(c["context"] + c["T"], dtype=torch.float64, device="cuda")
    angle = at[:, None] * freq[None, :]
    return torch.stack([torch.cos(angle) * length, torch.sin(angle) * length], dim=-1).float()


def _lengths(c):
    """Per sequence: its tokens in this call, and its tokens when the call is over (`attn`) or
    before it (`append`).  The batch's sum is the case's; which sequence has which is the seed's."""
    B, T = c["B"], c["T"]
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


def _batch(c, seed):
    new, have = _lengths(c)
    r = random.Random(seed)
    both = list(zip(new, have))
    r.shuffle(both)
    return [b[0] for b in both], [b[1] for b in both], r


def _pages(counts, r, prefix=None):
    """Page ids in the order of an allocator that has run for a while; -1 behind a sequence's last.
    prefix: how many of a sequence's first pages are those of one prompt that all began with."""
    prefix = prefix or [0] * len(counts)
    total = max(prefix) + sum(n - p for n, p in zip(counts, prefix))
    ids = list(range(total))
    r.shuffle(ids)
    common, ids = ids[:max(prefix)], ids[max(prefix):]
    rows, width = [], max(counts)
    for n, p in zip(counts, prefix):
        rows.append(common[:p] + [ids.pop() for _ in range(n - p)] + [-1] * (width - n))
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
    if c["kind"] == "rotary":
        x = _randn(g, c["T"], c["H"], c["D"]).to(DTYPES[c["dtype"]])
        at = torch.randint(0, c["context"], (c["T"],), generator=g, device="cuda", dtype=torch.int32)
        return dict(x=x, positions=at, table=_table(c))
    new, have, r = _batch(c, seed)
    page, block, D, H = c["page"], c["block"], c["D"], c["Hkv"]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    t = dict(cu=_int32(cu), have=_int32(have), most=max(new), longest=max(have))
    if c["kind"] == "append":
        counts = [-(-(n + h) // page) for n, h in zip(new, have)]
        t["pages"], total = _pages(counts, r, [h // page for h in have])
        t["k"], t["v"] = _new_rows(c, g)
        (t["kc"], t["ks"]), (t["vc"], t["vs"]) = [_codes(g, total, H, page, D, block) for _ in range(2)]
        t["table"] = _table(c) if c["rot"] else None
        return t
    t["pages"], total = _pages([-(-h // page) for h in have], r)
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
    if case["kind"] != "rotary" and case["T"] == case["B"]:
        s["cu"] = None  # one token each: the lengths of the chunks go without saying
    return s


# ------------------------------------------------------------- plain forms


def _rotate(x, table, positions, layout, offset, inverse=False):
    """fp32 [T, H, D] with the pairs of [offset, offset + rot) rotated."""
    cos, sin = table[positions.long()][:, None].unbind(-1)
    if inverse:
        sin = -sin
    rot = 2 * cos.shape[-1]
    y = x.float().clone()
    part = y[..., offset:offset + rot]
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
    c = s["case"]
    seq, at = _token_places(s)
    k = _rotate(s["k"], s["table"], at, c["layout"], 0) if c["rot"] else s["k"].float()
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
    if c["window"]:
        seen &= key > place[..., None] - c["window"]
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


def run(s):
    c = s["case"]
    if own:
        return _run_own(s)
    if c["kind"] == "rotary":
        return _rotate(s["x"], s["table"], s["positions"], c["layout"], c["offset"],
                       c["inverse"]).to(DTYPES[c["dtype"]])
    return _plain_append(s) if c["kind"] == "append" else _plain_attn(s)


_modules = []


def _run_own(s):
    c = s["case"]
    if not _modules:
        _package()
    R, P = _modules
    if c["kind"] == "rotary":
        return R.rotary(s["x"], s["table"], s["positions"], interleaved=c["layout"] == "interleaved",
                        offset=c["offset"], inverse=c["inverse"])
    cache = P.PagedKV(s["kc"], s["vc"], s["ks"], s["vs"])
    if c["kind"] == "append":
        P.append_kv(cache, s["k"], s["v"], s["pages"], s["have"], cu_tokens=s["cu"], table=s["table"],
                    interleaved=c["layout"] == "interleaved")
        return cache.k, cache.v, cache.k_scale, cache.v_scale
    return P.paged_attn(s["q"], cache, s["pages"], s["have"], cu_tokens=s["cu"], window=c["window"],
                        sink=s["sink"])


def _package():
    """The package's modules, imported by the first call with `own`."""
    at = os.path.join(os.getcwd(), "sglang-lite_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from sglang_lite_amd import paged_kv, rotary

    _modules[:] = [rotary, paged_kv]


# -------------------------------------------------------------------- work


def work(case):
    c = case
    if c["kind"] == "rotary":
        n = c["T"] * c["H"] * c["D"]
        size = 4 if c["dtype"] == "f32" else 2
        return dict(bytes=2 * n * size + c["T"] * (4 + 4 * c["rot"]), flops=3 * c["T"] * c["H"] * c["rot"])
    new, have = _lengths(c)
    H, D = c["Hkv"], c["D"]
    if c["kind"] == "append":
        n = c["T"] * H * D
        return dict(bytes=2 * n * 3 + c["T"] * 4 * c["rot"], flops=3 * c["T"] * H * c["rot"] + 4 * n)
    read = pairs = 0
    for n, h in zip(new, have):
        w = c["window"] or h
        read += min(h, n - 1 + w)
        full = min(n, max(0, h - w + 1)) if c["window"] else 0  # queries whose window is full
        part = n - full
        pairs += full * w + part * (h - n + 1) + part * (part - 1) // 2
    row = 2 * H * (D + 4 / c["block"])
    return dict(bytes=read * row + 4 * c["T"] * c["Hq"] * D, flops=4 * pairs * c["Hq"] * D)


# ------------------------------------------------------------------- exact


def _exact_rotated(c, x, at, layout, offset, inverse):
    """Rotation as a product of complex numbers, angles from the definition."""
    freq, length = _frequencies(c)
    turn = torch.polar(torch.full((at.numel(), 1, freq.numel()), length, dtype=torch.float64, device="cuda"),
                       (at.double()[:, None] * freq * (-1.0 if inverse else 1.0))[:, None])
    x = x.double()
    rot = c["rot"]
    head, part, tail = x[..., :offset], x[..., offset:offset + rot], x[..., offset + rot:]
    if layout == "half":
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * turn
        part = torch.cat([z.real, z.imag], dim=-1)
    else:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * turn
        part = torch.view_as_real(z).reshape(part.shape)
    return torch.cat([head, part, tail], dim=-1)


def _exact_append(c, t):
    """Sequence by sequence and block by block; codes before their rounding, as the values are then."""
    new, have = t["cu"].diff().tolist(), t["have"].tolist()
    page, block = c["page"], c["block"]
    pages = t["pages"].tolist()
    if c["rot"]:
        at = torch.cat([torch.arange(h, h + n, device="cuda") for n, h in zip(new, have)])
        k = _exact_rotated(c, t["k"], at, c["layout"], 0, False)
    else:
        k = t["k"].double()
    out = []
    for x, codes, scales in ((k, t["kc"], t["ks"]), (t["v"].double(), t["vc"], t["vs"])):
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
            for i0 in range(0, n, 1024):
                i1 = min(n, i0 + 1024)
                q = t["q"][row + i0:row + i1, j * G:(j + 1) * G].double()
                at = torch.arange(h - n + i0, h - n + i1, device="cuda")
                gap = at[:, None] - torch.arange(h, device="cuda")
                ok = (gap >= 0) & (gap < c["window"]) if c["window"] else gap >= 0
                for u in range(G):
                    e = (q[:, u] @ kt) * D ** -0.5
                    e = torch.where(ok, e, float("-inf"))
                    m = e.max(-1, keepdim=True).values.clamp_min(-1e300)
                    w = torch.exp(e - m)
                    den = w.sum(-1, keepdim=True)
                    if t["sink"] is not None:
                        den = den + torch.exp(t["sink"][j * G + u].double() - m)
                    o[row + i0:row + i1, j * G + u] = (w @ v) / den
        row += n
    return o


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    if c["kind"] == "rotary":
        return _exact_rotated(c, t["x"], t["positions"], c["layout"], c["offset"], c["inverse"])
    return _exact_append(c, t) if c["kind"] == "append" else _exact_attn(c, t)
