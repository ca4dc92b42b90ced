"""The operators between the q|k|v projection and the output projection of an attention layer
that keeps its keys and values in 8 bits with one scale for each block of tokens and head:

  norm_rope  norms of queries and keys for each head and the position rotation, in one pass
  update     new keys and values appended to the block-scaled cache, and the cache read back
  attend     attention of the newest tokens over the block-scaled cache
  step       one decode step of a layer: norm + rotation + append, then the attention

Each in a plain form (`own` false: elementary torch operations, fp32 inside) and through
llmquant_b200's public calls (`own` true). Shapes in the cases: batch sequences, `tokens` new
tokens each on top of `start` cached ones, hq query heads on hkv key/value heads of `dim` values,
`block` tokens to a scale. `ragged` sequences have different cached lengths and new-token counts.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode token of the 8B layer (32 query, 8 key heads of 128): latency of one launch
        dict(name="norm_rope decode", kind="norm_rope", batch=1, tokens=1, hq=32, hkv=8, dim=128, rot=128,
             norm=True, interleaved=False, dtype="bf16"),
        # a long prompt batch of the same layer: streaming
        dict(name="norm_rope prompts", kind="norm_rope", batch=4, tokens=8192, hq=32, hkv=8, dim=128, rot=128,
             norm=True, interleaved=False, dtype="bf16"),
        # odd token count and head counts, partial interleaved rotation, no norm, fp16
        dict(name="norm_rope odd", kind="norm_rope", batch=3, tokens=1237, hq=14, hkv=2, dim=64, rot=32,
             norm=False, interleaved=True, dtype="fp16"),
        # one token appended to a short conversation of the 1B layer (heads of 64) and the cache read
        dict(name="update token", kind="update", batch=1, tokens=1, start=99, hkv=8, dim=64, block=64,
             ragged=False, dtype="bf16"),
        # a prompt chunk with ragged counts on top of ragged cached lengths, small blocks
        dict(name="update ragged chunk", kind="update", batch=5, tokens=700, start=1600, hkv=4, dim=128, block=32,
             ragged=True, dtype="fp16"),
        # whole prompts into an empty cache, 8B heads: what a prefill does per layer
        dict(name="update prompts", kind="update", batch=8, tokens=4111, start=0, hkv=8, dim=128, block=64,
             ragged=False, dtype="bf16"),
        # a decode step at batch 1 on a 4k context, 8B heads
        dict(name="step batch 1", kind="step", batch=1, tokens=1, start=4110, hq=32, hkv=8, dim=128, block=64,
             norm=True, ragged=False, dtype="bf16"),
        # a decode step of 32 sequences of different lengths, 8B heads
        dict(name="step batch 32 ragged", kind="step", batch=32, tokens=1, start=4110, hq=32, hkv=8, dim=128, block=64,
             norm=True, ragged=True, dtype="bf16"),
        # one very long context: the work has to be split along it
        dict(name="attend long context", kind="attend", batch=1, tokens=1, start=131000, hq=32, hkv=8, dim=128, block=128,
             ragged=False, dtype="bf16"),
        # many ragged sequences with the 1B layer's heads
        dict(name="attend batch 64 ragged", kind="attend", batch=64, tokens=1, start=6001, hq=32, hkv=8, dim=64, block=64,
             ragged=True, dtype="bf16"),
        # five drafted tokens to verify per sequence, eight query heads to a key head, fp16
        dict(name="attend drafts", kind="attend", batch=8, tokens=5, start=2047, hq=16, hkv=2, dim=128, block=32,
             ragged=True, dtype="fp16"),
        # a prompt chunk read straight from the cache
        dict(name="attend chunk", kind="attend", batch=1, tokens=512, start=3499, hq=32, hkv=8, dim=128, block=64,
             ragged=False, dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("norm_rope", "update", "step", "attend"))
    dim = rng.choice((64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "norm_rope":
        hkv = rng.choice((1, 2, 4, 5, 8))
        hq = hkv * rng.choice((1, 2, 3, 4, 7))
        dim = rng.choice((64, 96, 128, 256))
        rot = rng.choice((dim, dim, dim // 2))
        batch = log(1, 32)
        tokens = min(log(1, 8192), max(1, 160_000_000 // (batch * (hq + hkv) * dim)))
        return dict(kind=kind, batch=batch, tokens=tokens, hq=hq, hkv=hkv, dim=dim, rot=rot,
                    norm=rng.random() < 0.7, interleaved=rng.random() < 0.3, dtype=dtype)
    block = rng.choice((16, 32, 64, 128))
    hkv = rng.choice((1, 2, 4, 8))
    ragged = rng.random() < 0.6
    if kind == "update":
        batch = log(1, 16)
        tokens = log(1, 4096)
        start = log(1, 4096)
        room = max(64, 33_000_000 // (batch * hkv * dim))
        tokens, start = min(tokens, room // 2), min(start, room // 2)
        if tokens > block:  # longer chunks begin where a block begins
            start -= start % block
        return dict(kind=kind, batch=batch, tokens=tokens, start=start, hkv=hkv, dim=dim, block=block,
                    ragged=ragged, dtype=dtype)
    hq = hkv * rng.choice((1, 2, 3, 4, 5, 7, 8))
    batch = log(1, 64)
    room = max(256, 130_000_000 // (batch * hkv * dim))
    start = min(log(16, 131000), room)
    if kind == "step":
        return dict(kind=kind, batch=batch, tokens=1, start=start, hq=hq, hkv=hkv, dim=dim, block=block,
                    norm=rng.random() < 0.7, ragged=ragged, dtype=dtype)
    tokens = 1 if rng.random() < 0.5 else log(2, 64)
    batch = batch if tokens == 1 else min(batch, 16)
    # (the plain form's score matrix bounds the context of many query rows)
    start = min(start, max(256, 1_000_000_000 // (batch * hq * tokens)))
    return dict(kind=kind, batch=batch, tokens=tokens, start=start, hq=hq, hkv=hkv, dim=dim, block=block,
                ragged=ragged, dtype=dtype)


# ------------------------------------------------------------------------------------- shapes
def _lengths(case):
    """Cached tokens and new tokens of each sequence (host integers). The first sequence is the longest."""
    batch, start, tokens, block = case["batch"], case["start"], case["tokens"], case["block"]
    if not case["ragged"]:
        return [start] * batch, [tokens] * batch
    starts = [start - (start * b) // (2 * batch) for b in range(batch)]
    if tokens > block:
        starts = [s - s % block for s in starts]
    counts = [tokens - (tokens * b) // (2 * batch) for b in range(batch)]
    return starts, counts


def _blocks(case):
    return -(-(case["start"] + case["tokens"]) // case["block"])


def work(case):
    es = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    d, t, b, hkv = case["dim"], case["tokens"], case["batch"], case["hkv"]
    if case["kind"] == "norm_rope":
        rows = b * t * (case["hq"] + hkv)
        # each value read and written once, each token's angles (cosine and sine of rot/2) once
        return {"bytes": 2 * rows * d * es + b * t * (case["rot"] * 4 + 8), "flops": rows * d * 7}
    starts, counts = _lengths(case)
    block, hq = case["block"], case.get("hq", 0)
    total = flops = 0
    for s, n in zip(starts, counts):
        length = s + n
        full, tail = length - length % block, length % block
        held = 2 * hkv * (full * d + full // block * 4)  # codes and scales of the complete blocks
        new = 2 * hkv * n * d * es
        if case["kind"] == "update":
            old = 2 * hkv * ((s - s % block) * d + s // block * 4)
            fresh = held - old
            total += new + max(fresh, 0) + old + 2 * hkv * max(tail - n, 0) * d * es + 2 * hkv * min(n, 2 * block) * d * es
            total += 2 * hkv * length * d * es  # what is read back, written out
            flops += 2 * hkv * (length + n) * d * 2
            continue
        total += held + 2 * hkv * tail * d * es + 2 * n * hq * d * es
        if case["kind"] == "step":
            total += 2 * new + n * hq * d * es + d * 4
        seen = sum(s + i + 1 for i in range(n))
        flops += 4 * hq * d * seen
    return {"bytes": total, "flops": flops}


# ------------------------------------------------------------------------------------- inputs
def _tables(length, rot, device):
    """cos and sin of position * 500000^(-2 i / rot), angles in 64 bits, tables in 32."""
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _cache(case, gen):
    """A block-scaled cache as it stands after `start` tokens of each sequence, its pages scattered over the pool."""
    dev, dt = "cuda", DTYPES[case["dtype"]]
    b, h, d, p, nb = case["batch"], case["hkv"], case["dim"], case["block"], _blocks(case)
    pages = b * nb
    table = torch.randperm(pages, generator=gen, device=dev).reshape(b, nb).to(torch.int32)
    s = {"table": table}
    for name in "kv":
        # keys have channels of different size, values less so
        size = torch.rand(h, 1, d, generator=gen, device=dev) * (2.0 if name == "k" else 0.5) + 0.5
        codes = torch.empty(pages, h, p, d, dtype=torch.int8, device=dev)
        scales = torch.empty(pages, h, dtype=torch.float32, device=dev)
        for lo in range(0, pages, 4096):
            x = torch.randn(min(4096, pages - lo), h, p, d, generator=gen, device=dev) * size
            scale = (x.abs().amax((2, 3)) / 127).clamp_min(1e-8)
            scales[lo:lo + 4096] = scale
            codes[lo:lo + 4096] = (x / scale[..., None, None]).round().clamp(-128, 127).to(torch.int8)
        s[name + "_pages"], s[name + "_scales"] = codes, scales
        s[name + "_ring"] = (torch.randn(b, h, 2 * p, d, generator=gen, device=dev) * size).to(dt)
    starts, counts = _lengths(case)
    s["start"] = torch.tensor(starts, dtype=torch.int64).to(dev)
    s["count"] = torch.tensor(counts, dtype=torch.int64).to(dev)
    if own:  # the handle that a program keeps for a layer's cache
        from llmquant_b200.quantizers import BlockKVStore

        s["store"] = BlockKVStore(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["k_ring"], s["v_ring"],
                                  s["table"])
    return s


def prepare(case, seed):
    dev, dt = "cuda", DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    b, t, h, d = case["batch"], case["tokens"], case["hkv"], case["dim"]
    kind = case["kind"]
    s = {"case": dict(case)}
    if kind == "norm_rope":
        hq = case["hq"]
        qkv = torch.randn(b, t, hq + 2 * h, d, generator=gen, device=dev) * 1.5
        s["qkv"] = qkv.to(dt)  # the fused projection's output; q and k are its first heads
        table_len = 16384
        first = torch.randint(0, table_len - t, (b, 1), generator=gen, device=dev)
        s["positions"] = first + torch.arange(t, device=dev)
        s["cos"], s["sin"] = _tables(table_len, case["rot"], dev)
        if case["norm"]:
            s["q_weight"] = (torch.rand(d, generator=gen, device=dev) + 0.5).to(dt)
            s["k_weight"] = (torch.rand(d, generator=gen, device=dev) + 0.5).to(dt)
        return s
    s.update(_cache(case, gen))
    if kind == "update":
        # as attention layers hand them over: [batch, tokens, heads, dim] seen with the heads in front
        s["k_new"] = torch.randn(b, t, h, d, generator=gen, device=dev).to(dt).transpose(1, 2)
        s["v_new"] = torch.randn(b, t, h, d, generator=gen, device=dev).to(dt).transpose(1, 2)
    elif kind == "step":
        s["qkv"] = (torch.randn(b, t, case["hq"] + 2 * h, d, generator=gen, device=dev) * 1.5).to(dt)
        s["cos"], s["sin"] = _tables(case["start"] + t, d, dev)
        if case["norm"]:
            s["q_weight"] = (torch.rand(d, generator=gen, device=dev) + 0.5).to(dt)
            s["k_weight"] = (torch.rand(d, generator=gen, device=dev) + 0.5).to(dt)
    else:
        s["q"] = (torch.randn(b, t, case["hq"], d, generator=gen, device=dev) * 1.5).to(dt)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _norm_rope(x, weight, cos, sin, interleaved, eps):
    """fp32 [.., heads, D] from x [.., heads, D]; cos, sin [.., 1, rot/2]; not rounded."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()
    half = cos.shape[-1]
    turn, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, c = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack((a * cos - c * sin, c * cos + a * sin), -1).flatten(-2)
    else:
        a, c = turn[..., :half], turn[..., half:]
        turned = torch.cat((a * cos - c * sin, c * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _run_norm_rope(s):
    case = s["case"]
    hq, h = case["hq"], case["hkv"]
    q, k = s["qkv"][:, :, :hq], s["qkv"][:, :, hq:hq + h]
    if own:
        from llmquant_b200.cuda import qk_norm_rope

        q, k = qk_norm_rope(q, k, s["cos"], s["sin"], s["positions"], q_weight=s.get("q_weight"),
                            k_weight=s.get("k_weight"), eps=1e-6, interleaved=case["interleaved"])
        return {"q": q, "k": k}
    cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
    return {name: _norm_rope(x, s.get(name + "_weight"), cos, sin, case["interleaved"], 1e-6).to(x.dtype)
            for name, x in (("q", q), ("k", k))}


def _held(s, name, block):
    """fp32 values of every block of a sequence's pages, [B, H, blocks * P, D]."""
    pages = s["table"].long()
    x = s[name + "_pages"][pages].float() * s[name + "_scales"][pages][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _ring_values(s, name, block, blocks):
    """The ring's rows at the positions of the last two blocks of `total`, spread over all positions."""
    slots = torch.arange(blocks * block, device="cuda") % (2 * block)
    return s[name + "_ring"][:, :, slots]


def _append(s, name, new, case):
    """The new rows written into the cache's own buffers, blocks that are complete now quantised."""
    block, blocks, t = case["block"], _blocks(case), case["tokens"]
    b, h, d = case["batch"], case["hkv"], case["dim"]
    start, total = s["start"][:, None], (s["start"] + s["count"])[:, None]
    pos = torch.arange(blocks * block, device="cuda")[None]
    fresh = (pos >= start) & (pos < total)
    at = (pos - start).clamp(0, t - 1)
    rows = new.gather(2, at[:, None, :, None].expand(b, h, blocks * block, d))
    raw = torch.where(fresh[:, None, :, None], rows, _ring_values(s, name, block, blocks)).float()
    raw = raw.reshape(b, h, blocks, block, d)
    number = torch.arange(blocks, device="cuda")[None]
    done = (number >= start // block) & (number < total // block)  # became complete in this call
    scale = (raw.abs().amax((3, 4)) / 127).clamp_min(1e-8)
    codes = (raw / scale[..., None, None]).round().clamp(-128, 127).to(torch.int8)
    pages = s["table"].long()
    keep = done[:, :, None]
    s[name + "_pages"][pages] = torch.where(keep[..., None, None], codes.permute(0, 2, 1, 3, 4), s[name + "_pages"][pages])
    s[name + "_scales"][pages] = torch.where(keep, scale.transpose(1, 2), s[name + "_scales"][pages])
    # ring: slot -> the position of the last two blocks that it belongs to
    slot = torch.arange(2 * block, device="cuda")[None]
    last = total // block
    own_block = torch.where((last % 2) == slot // block, last, last - 1)
    where = own_block * block + slot % block
    fresh = (where >= start) & (where < total)
    at = (where - start).clamp(0, t - 1)
    rows = new.gather(2, at[:, None, :, None].expand(b, h, 2 * block, d))
    ring = s[name + "_ring"]
    ring.copy_(torch.where(fresh[:, None, :, None], rows, ring))


def _values(s, name, case):
    """fp32 [B, H, positions, D]: what the cache stands for after the call's tokens, zeros behind them."""
    block, blocks = case["block"], _blocks(case)
    total = (s["start"] + s["count"])[:, None]
    pos = torch.arange(blocks * block, device="cuda")[None]
    complete = (pos < total // block * block)[:, None, :, None]
    x = torch.where(complete, _held(s, name, block), _ring_values(s, name, block, blocks).float())
    return torch.where((pos < total)[:, None, :, None], x, torch.zeros((), device="cuda"))


def _run_update(s):
    case = s["case"]
    length = case["start"] + case["tokens"]
    if own:
        store = s["store"]
        store.append(s["k_new"], s["v_new"], s["start"], s["count"])
        k, v = store.read(length, s["start"], s["count"])
        return {"k": k, "v": v, "k_ring": store.k_ring, "v_ring": store.v_ring}
    out = {}
    for name in "kv":
        _append(s, name, s[name + "_new"], case)
        out[name] = _values(s, name, case)[:, :, :length].to(s[name + "_new"].dtype)
        out[name + "_ring"] = s[name + "_ring"]
    return out


def _attend(q, s, case):
    b, t, h, d = case["batch"], case["tokens"], case["hkv"], case["dim"]
    group = case["hq"] // h
    k, v = _values(s, "k", case), _values(s, "v", case)
    rows = q.float().reshape(b, t, h, group, d).permute(0, 2, 1, 3, 4).reshape(b, h, t * group, d)
    scores = (rows @ k.transpose(2, 3)) * d ** -0.5
    pos = torch.arange(k.shape[2], device="cuda")
    new = torch.arange(t, device="cuda")
    seen = (pos[None, None] <= (s["start"][:, None] + new)[..., None]) & (new[None] < s["count"][:, None])[..., None]
    seen = seen[:, None].repeat_interleave(group, 2)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    whole = weights.sum(-1, keepdim=True)
    out = (weights @ v) / torch.where(whole == 0, torch.ones((), device="cuda"), whole)
    return out.reshape(b, h, t, group, d).permute(0, 2, 1, 3, 4).reshape(b, t, h * group, d).to(q.dtype)


def _run_attend(s):
    case = s["case"]
    if own:
        return s["store"].attend(s["q"], s["start"], s["count"])
    return _attend(s["q"], s, case)


def _run_step(s):
    case = s["case"]
    hq, h = case["hq"], case["hkv"]
    if own:
        store = s["store"]
        q = store.append_qkv(s["qkv"], s["cos"], s["sin"], s["start"], s["count"], q_weight=s.get("q_weight"),
                             k_weight=s.get("k_weight"), eps=1e-6)
        out = store.attend(q, s["start"], s["count"])
        return {"q": q, "out": out, "k_ring": store.k_ring, "v_ring": store.v_ring}
    pos = s["start"][:, None] + torch.arange(case["tokens"], device="cuda")
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    q, k, v = s["qkv"].split((hq, h, h), 2)
    q = _norm_rope(q, s.get("q_weight"), cos, sin, False, 1e-6).to(q.dtype)
    k = _norm_rope(k, s.get("k_weight"), cos, sin, False, 1e-6).to(q.dtype)
    _append(s, "k", k.transpose(1, 2), case)
    _append(s, "v", v.transpose(1, 2), case)
    return {"q": q, "out": _attend(q, s, case), "k_ring": s["k_ring"], "v_ring": s["v_ring"]}


def run(state):
    return {"norm_rope": _run_norm_rope, "update": _run_update, "attend": _run_attend,
            "step": _run_step}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------- 64 bits
def _turn64(x, weight, cos, sin, interleaved):
    """One token's heads [heads, D] in 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * weight.double()
    out = x.clone()
    half = cos.shape[-1]
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    out[..., first] = x[..., first] * cos.double() - x[..., second] * sin.double()
    out[..., second] = x[..., second] * cos.double() + x[..., first] * sin.double()
    return out


class _Sequence64:
    """One sequence's cache in 64 bits: complete blocks quantised from the values that arrived."""

    def __init__(self, s, name, b, case):
        self.block, start = case["block"], int(s["start"][b])
        whole = start // self.block
        pages = s["table"][b, :whole].long()
        held = s[name + "_pages"][pages].double() * s[name + "_scales"][pages].double()[:, :, None, None]
        self.done = [held.transpose(0, 1).reshape(case["hkv"], whole * self.block, case["dim"])]
        base = (whole % 2) * self.block
        self.open = s[name + "_ring"][b, :, base:base + start % self.block].double()

    def append(self, rows):
        """rows [H, n, D]"""
        rows = torch.cat((self.open, rows.double()), 1)
        whole = rows.shape[1] // self.block
        x = rows[:, : whole * self.block].unflatten(1, (whole, self.block))
        scale = (x.abs().amax((2, 3), keepdim=True) / 127).clamp_min(1e-8) if whole else x.new_ones(x.shape[0], 0, 1, 1)
        self.done.append(((x / scale).round().clamp(-128, 127) * scale).flatten(1, 2))
        self.open = rows[:, whole * self.block:]

    def values(self):
        return torch.cat((*self.done, self.open), 1)


def _ring64(s, name, b, rows, case):
    """The ring of sequence b after rows [H, n, D] at its start, in 64 bits."""
    ring, start = s[name + "_ring"][b].double(), int(s["start"][b])
    total = start + rows.shape[1]
    lowest = max(start, (total // case["block"] - 1) * case["block"])
    at = torch.arange(lowest, total, device="cuda")
    ring[:, at % (2 * case["block"])] = rows.double()[:, at - start]
    return ring


def _attend64(q, k, v, start):
    """q [n, Hq, D] at positions start .. start + n - 1 over k, v [H, start + n, D]."""
    n, hq, d = q.shape
    group = hq // k.shape[0]
    rows = q.double().permute(1, 0, 2).unflatten(0, (k.shape[0], group))
    scores = torch.einsum("hgnd,hld->hgnl", rows, k) / math.sqrt(d)
    ahead = torch.arange(k.shape[1], device="cuda")[None] > start + torch.arange(n, device="cuda")[:, None]
    prob = torch.softmax(scores.masked_fill(ahead, -math.inf), -1)
    return torch.einsum("hgnl,hld->hgnd", prob, v).flatten(0, 1).permute(1, 0, 2)


def exact(case, seed):
    s = prepare(case, seed)
    b, t, h, d = case["batch"], case["tokens"], case["hkv"], case["dim"]
    if case["kind"] == "norm_rope":
        cos, sin = s["cos"][s["positions"]][:, :, None], s["sin"][s["positions"]][:, :, None]
        hq = case["hq"]
        return {"q": _turn64(s["qkv"][:, :, :hq], s.get("q_weight"), cos, sin, case["interleaved"]),
                "k": _turn64(s["qkv"][:, :, hq:hq + h], s.get("k_weight"), cos, sin, case["interleaved"])}
    starts, counts = _lengths(case)
    length = case["start"] + t
    if case["kind"] == "update":
        out = {n: torch.zeros(b, h, length, d, dtype=torch.float64, device="cuda") for n in "kv"}
        for n in "kv":
            ring = []
            for i in range(b):
                seq = _Sequence64(s, n, i, case)
                rows = s[n + "_new"][i, :, : counts[i]]
                seq.append(rows)
                out[n][i, :, : starts[i] + counts[i]] = seq.values()
                ring.append(_ring64(s, n, i, rows, case))
            out[n + "_ring"] = torch.stack(ring)
        return out
    hq = case["hq"]
    out = torch.zeros(b, t, hq, d, dtype=torch.float64, device="cuda")
    extra = {"q": torch.zeros_like(out), "k_ring": [], "v_ring": []}
    for i in range(b):
        n = counts[i]
        k, v = _Sequence64(s, "k", i, case), _Sequence64(s, "v", i, case)
        if case["kind"] == "step":
            pos = starts[i] + torch.arange(n, device="cuda")
            cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
            extra["q"][i, :n] = _turn64(s["qkv"][i, :n, :hq], s.get("q_weight"), cos, sin, False)
            # queries and keys are held in the cache's type: one rounding each, as the operator defines
            q = extra["q"][i, :n].to(DTYPES[case["dtype"]])
            rows_k = _turn64(s["qkv"][i, :n, hq:hq + h], s.get("k_weight"), cos, sin, False).transpose(0, 1)
            rows_v = s["qkv"][i, :n, hq + h:].transpose(0, 1)
            extra["k_ring"].append(_ring64(s, "k", i, rows_k, case))
            extra["v_ring"].append(_ring64(s, "v", i, rows_v, case))
            k.append(rows_k.to(DTYPES[case["dtype"]]))
            v.append(rows_v)
            k, v = k.values(), v.values()
        else:
            q = s["q"][i, :n]
            k, v = (_held64(s, m, i, starts[i] + n, case) for m in "kv")
        out[i, :n] = _attend64(q, k, v, starts[i])
    if case["kind"] == "attend":
        return out
    return {"q": extra["q"], "out": out, "k_ring": torch.stack(extra["k_ring"]), "v_ring": torch.stack(extra["v_ring"])}


def _held64(s, name, b, total, case):
    """Sequence b's values in 64 bits when all `total` tokens are in the cache already."""
    block = case["block"]
    whole = total // block
    pages = s["table"][b, :whole].long()
    held = s[name + "_pages"][pages].double() * s[name + "_scales"][pages].double()[:, :, None, None]
    base = (whole % 2) * block
    return torch.cat((held.transpose(0, 1).flatten(1, 2), s[name + "_ring"][b, :, base:base + total % block].double()), 1)
