"""What the cached-attention operators are measured on: rotary positions, appending keys and values to a
paged cache held in 4 bits (with the keys' rotation applied on the way), and attention over that cache.

The cache's layout, in the plain form's tensors as in the operators' storages (P pages of S slots, H heads
of D channels, groups of 32 channels):
  k codes   [P, H, S, D % 32 / 8, D / 32, D % 8]  signed 4-bit, two to a byte, the low nibble first
  v codes   [P, H, S, D % 32 / 4, D / 32, D % 4]
  scales    [P, H, S, D / 32, 2]                  bf16 (step, offset) of each group, for k and for v
A stored value is code * step + offset.
"""
import math

import torch

own = False

GROUP = 32  # channels that share a step and an offset
MOST64 = 10 ** 14  # multiplications that the form in 64 bits takes on


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def _rotary(name, tokens, heads, dim, rot, layout, dtype, scaling, far, extra=0):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "dim": dim, "rot": rot,
            "layout": layout, "dtype": dtype, "scaling": scaling, "far": far, "extra": extra}


def _append(name, tokens, heads, dim, rot, layout, dtype, scaling, far, page, pages, skipped):
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "dim": dim, "rot": rot,
            "layout": layout, "dtype": dtype, "scaling": scaling, "far": far, "page": page, "pages": pages,
            "skipped": skipped}


def _attend(name, q, kv, heads, group, dim, page, causal=True):
    return {"name": name, "op": "attention", "q": ",".join(map(str, q)), "kv": ",".join(map(str, kv)),
            "heads": heads, "group": group, "dim": dim, "page": page, "causal": causal}


def listed():
    ragged = [64 + (b * 40503 + 977) % 8129 for b in range(64)]
    return [
        # one new token of one user: the queries of a 32-head block, latency alone
        _rotary("rotary_token", 1, 32, 128, 128, "half", "bf16", "none", 8192),
        # the queries of 8 prompts of 512 tokens (the decoder block's own shape), positions stretched by parts
        _rotary("rotary_prompts", 4096, 32, 128, 128, "half", "bf16", "by_parts", 131072),
        # two thirds of each head rotated, neighbouring pairs, read out of a wider row, far positions
        _rotary("rotary_partial", 1025, 20, 96, 64, "interleaved", "f32", "linear", 1000000, 480),
        # one new token of each of 64 users
        _append("append_tokens", 64, 8, 128, 128, "half", "bf16", "none", 8192, 16, 80, 0),
        # 8 prompts of 512 tokens into pages of 64
        _append("append_prompts", 4096, 8, 128, 128, "half", "bf16", "by_parts", 131072, 64, 72, 0),
        # a padded batch: 100 of its rows are no tokens; f32 projections, smaller heads, a part rotated
        _append("append_padded", 1001, 3, 64, 32, "interleaved", "f32", "ntk", 32768, 32, 40, 100),
        # one user's next token, early in an answer: latency
        _attend("attention_token", [1], [777], 8, 4, 128, 16),
        # the next token of 64 users of all lengths
        _attend("attention_batch", [1] * 64, ragged, 8, 4, 128, 16),
        # the next token of two long contexts
        _attend("attention_long", [1, 1], [131072, 100003], 8, 4, 128, 64),
        # the next 512 tokens of long prompts taken in pieces
        _attend("attention_pieces", [512] * 4, [4096, 2048, 3585, 512], 8, 4, 128, 64),
        # 8 whole prompts of 512 tokens
        _attend("attention_prompts", [512] * 8, [512] * 8, 8, 4, 128, 64),
        # pieces and single tokens mixed, one sequence without new tokens, one with fewer keys than queries,
        # small heads that seven query heads share
        _attend("attention_mixed", [1, 37, 0, 130, 5, 1], [1025, 37, 640, 1999, 3, 0], 3, 7, 64, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention"])
    scaling, layout = rng.choice(["none", "linear", "ntk", "by_parts"]), rng.choice(["half", "interleaved"])
    dtype, far = rng.choice(["bf16", "f32"]), _log(rng, 16, 1000000)
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 160, 256])
        heads = rng.randint(1, 40)
        tokens = _log(rng, 1, 4096 * 4096 // (heads * dim) // (2 if dtype == "f32" else 1))
        rot = rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        return _rotary("", min(tokens, 20000), heads, dim, rot, layout, dtype, scaling, far,
                       rng.choice([0, 0, 8 * rng.randint(1, 64)]))
    if op == "append":
        dim, heads, page = rng.choice([64, 128, 256]), rng.randint(1, 8), rng.choice([16, 32, 64, 128])
        tokens = _log(rng, 1, min(6000, 4096 * 1024 // (heads * dim)))
        rot = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        return _append("", tokens, heads, dim, rot, layout, dtype, scaling, far, page,
                       -(-tokens // page) + rng.randint(1, 4), rng.choice([0, 0, tokens // 7]))
    dim, heads, group = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8, 12])
    page = rng.choice([16, 32, 64, 128])
    if rng.random() < 0.5:  # single tokens
        longest = _log(rng, 1, 131072)
        most = min(64, 262144 // longest, 2 ** 28 // (longest * heads * dim))
        kv = [rng.randint(1, longest) for _ in range(_log(rng, 1, max(1, most)))]
        kv[-1] = longest
        q = [1] * len(kv)
    else:  # pieces of prompts, with single tokens among them
        longest = _log(rng, 16, 4096)
        most = max(1, min(8, 2 ** 23 * 32 // (longest * min(longest, 512) * heads * group)))
        kv = [rng.randint(1, longest) for _ in range(rng.randint(1, most))]
        q = [min(512, rng.choice([1, n, rng.randint(0, n)])) for n in kv]
        q[0] = max(1, q[0])
    return _attend("", q, kv, heads, group, dim, page, rng.random() < 0.85)


def _whole(text):
    return [int(x) for x in text.split(",")]


# ---------------------------------------------------------------------------------------------
# what every form starts from
# ---------------------------------------------------------------------------------------------
def _frequencies(case):
    """The rotation's angle per position of each pair, in 64 bits, and what the rotated part is scaled by."""
    n = case["rot"] // 2
    i = torch.arange(n, dtype=torch.float64)
    base = 500000.0
    if case["scaling"] == "ntk":  # a factor of 4 through the base
        base *= 4.0 ** (case["rot"] / max(case["rot"] - 2, 1))
    f = base ** (-2.0 * i / case["rot"])
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "by_parts":  # by the turns that a pair makes over the 8192 positions first learned
        keep = ((8192.0 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return f / 16.0 * (1 - keep) + f * keep, 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _noise(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _positions(gen, case):
    # runs of neighbouring positions, as sequences have them, from places all over the range
    t = torch.arange(case["tokens"], device="cuda")
    start = torch.randint(0, max(1, case["far"]), (case["tokens"] // 64 + 1,), generator=gen, device="cuda")
    return ((start[t // 64] + t % 64) % max(1, case["far"])).to(torch.int32)


def _quantised(x):
    """x [..., D] -> codes [..., D / 32, 32], steps and offsets [..., D / 32] bf16. In the arithmetic of
    x: 64 bits where its codes are compared, since a value next to a border takes the one or the other."""
    g = x.unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    step = ((hi - lo) / 15.0).float().bfloat16()
    offset = (lo + 8.0 * step.to(x.dtype)).float().bfloat16()
    by = torch.where(step > 0, step.to(x.dtype), math.inf)
    return ((g - offset.to(x.dtype)[..., None]) / by[..., None]).round().clamp(-8, 7), step, offset


def _packed(codes, width):
    """codes [..., D / 32, 32] -> bytes [..., D / 2] in the order [D % 32 / width, D / 32, D % width]."""
    c = codes.to(torch.int32).unflatten(-1, (-1, width)).transpose(-3, -2).flatten(-3) & 15
    return (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8)


def _unpacked(data, scales, width):
    """bytes [..., D / 2] and scales [..., D / 32, 2] -> values [..., D] f32."""
    c = torch.stack([data & 15, data >> 4], -1).flatten(-2).to(torch.int32)
    c = torch.where(c > 7, c - 16, c).unflatten(-1, (GROUP // width, -1, width)).transpose(-3, -2).flatten(-2).float()
    return (c * scales[..., 0, None].float() + scales[..., 1, None].float()).flatten(-2)


def _cache(gen, pages, heads, page, dim):
    """Pages full of keys and values: channels of different sizes and means, as projections give them."""
    k = _noise(gen, pages, heads, page, dim) * (0.5 + _noise(gen, heads, 1, dim).abs()) + _noise(gen, heads, 1, dim)
    v = _noise(gen, pages, heads, page, dim) + 0.2 * _noise(gen, heads, 1, dim)
    kc, ks, ko = _quantised(k)
    vc, vs, vo = _quantised(v)
    return {"k": _packed(kc, 8), "v": _packed(vc, 4), "k_scale": torch.stack([ks, ko], -1),
            "v_scale": torch.stack([vs, vo], -1)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "attention":
        q, kv, page = _whole(case["q"]), _whole(case["kv"]), case["page"]
        need = [-(-n // page) for n in kv]
        width, pages = max(1, max(need)), sum(need) + 3
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        slot = torch.arange(width, device="cuda")[None]
        need_t = torch.tensor(need, device="cuda")
        first = need_t.cumsum(0) - need_t
        s["table"] = torch.where(slot < need_t[:, None], order[(first[:, None] + slot).clamp(max=pages - 1)], -1)
        s["q_start"] = torch.tensor([0] + q, device="cuda").cumsum(0).to(torch.int32)
        s["kv_len"] = torch.tensor(kv, device="cuda", dtype=torch.int32)
        s["cache"] = _cache(gen, pages, case["heads"], page, case["dim"])
        s["q"] = _noise(gen, sum(q), case["heads"] * case["group"], case["dim"]).bfloat16()
        # the sequence of each query token and its place there, as a padded batch is built from
        s["of"] = torch.repeat_interleave(torch.arange(len(q), device="cuda"), torch.tensor(q, device="cuda"))
        s["at"] = torch.arange(sum(q), device="cuda") - s["q_start"][:-1].long()[s["of"]]
    else:
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        freq, size = _frequencies(case)
        s["freq"], s["size"], s["positions"] = freq.cuda(), size, _positions(gen, case)
        row = (case["tokens"], case["heads"], case["dim"])
        if case["op"] == "rotary":  # one part of a row that a fused projection wrote
            s["row"] = _noise(gen, case["tokens"], case["heads"] * case["dim"] + case["extra"]).to(dtype)
            s["x"] = s["row"][:, case["extra"]:].view(row)
        else:
            bias = _noise(gen, case["heads"], case["dim"])
            s["k"], s["v"] = (_noise(gen, *row) + bias).to(dtype), _noise(gen, *row).to(dtype)
            slots = torch.randperm(case["pages"] * case["page"], generator=gen, device="cuda")[:case["tokens"]]
            skip = torch.randperm(case["tokens"], generator=gen, device="cuda")[:case["skipped"]]
            slots[skip] = -1
            s["slots"] = slots.to(torch.int32)
            s["written"] = (slots >= 0).nonzero()[:, 0]
            s["cache"] = _cache(gen, case["pages"], case["heads"], case["page"], case["dim"])
    if own:
        _hold(s, case)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------------------------
def _rotated(x, s, case):
    """x [T, H, D]: each pair turned by its token's angle, the angle in 64 bits."""
    turn = s["positions"].double()[:, None] * s["freq"]
    c, n = (turn.cos() * s["size"]).to(x.dtype)[:, None], (turn.sin() * s["size"]).to(x.dtype)[:, None]
    rot = case["rot"]
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _plain_append(s, case):
    cache, page, rows = s["cache"], case["page"], s["written"]
    slots = s["slots"][rows].long()
    for name, x, width in (("k", _rotated(s["k"].double(), s, case), 8), ("v", s["v"].double(), 4)):
        codes, step, offset = _quantised(x[rows])
        cache[name][slots // page, :, slots % page] = _packed(codes, width)
        cache[name + "_scale"][slots // page, :, slots % page] = torch.stack([step, offset], -1)
    return {n: _unpacked(cache[n], cache[n + "_scale"], w).transpose(1, 2).flatten(0, 1).bfloat16().contiguous()
            for n, w in (("k", 8), ("v", 4))}


def _plain_attention(s, case):
    cache, page, group, dim = s["cache"], case["page"], case["group"], case["dim"]
    table = s["table"].clamp(min=0).long()
    batch, keys = table.shape[0], table.shape[1] * page
    k = _unpacked(cache["k"][table], cache["k_scale"][table], 8).transpose(1, 2).flatten(2, 3)  # [B, H, keys, D]
    v = _unpacked(cache["v"][table], cache["v_scale"][table], 4).transpose(1, 2).flatten(2, 3)
    longest = max(_whole(case["q"]))
    q = torch.zeros(batch, longest, case["heads"], group, dim, device="cuda")
    q[s["of"], s["at"]] = s["q"].float().unflatten(1, (case["heads"], group))
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, H, group * longest, D]
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(dim ** -0.5)
    count = s["q_start"].diff()[:, None]
    last = s["kv_len"][:, None].expand(batch, longest)  # the first key that a query does not see
    if case["causal"]:
        last = last - count + torch.arange(1, longest + 1, device="cuda")
    seen = torch.arange(keys, device="cuda") < last[..., None]  # [B, longest, keys]
    seen = seen[:, None, None].expand(batch, 1, group, longest, keys).flatten(2, 3)
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, torch.where((torch.arange(keys, device="cuda") < s["kv_len"][:, None])[:, None, :, None], v, 0.0))
    o = torch.where(total > 0, o / total, 0.0)
    o = o.unflatten(2, (group, longest)).permute(0, 3, 1, 2, 4)  # [B, longest, H, group, D]
    return o[s["of"], s["at"]].flatten(1, 2).bfloat16()


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "rotary":
        return _rotated(state["x"].float(), state, case).to(state["x"].dtype)
    if case["op"] == "append":
        return _plain_append(state, case)
    return _plain_attention(state, case)


# ---------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------
class _Memory:
    """A storage's device memory for torch (no copy; a tensor over it keeps the storage)."""

    def __init__(self, storage, shape, kind):
        self.storage = storage
        self.__cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (storage.addr, False), "version": 3}


def _tensor(storage, shape):
    if storage.dtype == "bf16":
        return torch.as_tensor(_Memory(storage, shape, "<i2"), device="cuda").view(torch.bfloat16)
    return torch.as_tensor(_Memory(storage, shape, "<f4"), device="cuda")


_KEPT = {}


def _backend():
    if not _KEPT:
        import __graft_entry__
        fb = __graft_entry__._pkg()
        _KEPT["fb"], _KEPT["be"] = fb, fb.B200(torch.cuda.current_device())
    be = _KEPT["be"]
    be.set_stream(torch.cuda.current_stream().cuda_stream)
    return _KEPT["fb"], be


def _copied(fb, be, x, dtype):
    """A storage with a tensor's values."""
    s = fb.Storage(be, dtype, x.numel() * (2 if dtype == "i4" else 1), zero=False)
    x = x.contiguous()
    _tensor_bytes(s).copy_(x.view(-1).view(torch.uint8))
    return s


def _tensor_bytes(storage):
    return torch.as_tensor(_Memory(storage, (storage.nbytes,), "|u1"), device="cuda")


def _hold(s, case):
    """The storages and handles that a user's program keeps."""
    fb, be = _backend()
    h = s["held"] = {}
    if case["op"] == "attention":
        h["q"] = _copied(fb, be, s["q"], "bf16")
        h["out"] = fb.Storage(be, "bf16", s["q"].numel())
        h["seen"] = _tensor(h["out"], tuple(s["q"].shape))
        for name in ("table", "q_start", "kv_len"):
            h[name] = _copied(fb, be, s[name], "i32")
    else:
        h["positions"] = _copied(fb, be, s["positions"], "i32")
        h["rope"] = fb.Rope(s["freq"].cpu().tolist(), layout=case["layout"], magnitude=s["size"])
        if case["op"] == "rotary":
            h["row"] = _copied(fb, be, s["row"], case["dtype"])
            h["out"] = fb.Storage(be, case["dtype"], s["x"].numel())
            h["seen"] = _tensor(h["out"], tuple(s["x"].shape))
        else:
            for name in ("k", "v"):
                h[name] = _copied(fb, be, s[name], case["dtype"])
            h["slots"] = _copied(fb, be, s["slots"], "i32")
            slots = case["pages"] * case["page"]
            h["all"] = _copied(fb, be, torch.arange(slots, device="cuda", dtype=torch.int32), "i32")
            h["out"] = [fb.Storage(be, "bf16", slots * case["heads"] * case["dim"]) for _ in range(2)]
            h["seen"] = {n: _tensor(o, (slots, case["heads"], case["dim"])) for n, o in zip("kv", h["out"])}
    if case["op"] != "rotary":
        pages = s["cache"]["k"].shape[0]
        h["cache"] = fb.PagedCache(be, pages, case["page"], case["heads"], case["dim"])
        for name in ("k", "v", "k_scale", "v_scale"):
            _tensor_bytes(getattr(h["cache"], name)).copy_(s["cache"][name].view(-1).view(torch.uint8))


def _own(s, case):
    _, be = _backend()
    h = s["held"]
    if case["op"] == "rotary":
        be.rotary(h["row"], h["positions"], h["rope"], case["heads"], case["dim"], out=h["out"],
                  x_offset=case["extra"], x_stride=case["heads"] * case["dim"] + case["extra"])
    elif case["op"] == "append":
        be.cache_append(h["cache"], h["k"], h["v"], h["slots"], positions=h["positions"], rope=h["rope"])
        be.cache_read(h["cache"], h["all"], out=h["out"])
    else:
        be.cache_attention(h["q"], h["cache"], h["table"], h["q_start"], h["kv_len"], case["heads"] * case["group"],
                           causal=case["causal"], out=h["out"])
    return h["seen"]


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without, and the values in 64 bits
# ---------------------------------------------------------------------------------------------
def work(case):
    dim, heads = case["dim"], case["heads"]
    stored = heads * 2 * (dim // 2 + dim // GROUP * 4)  # bytes of one token's keys and values
    if case["op"] == "rotary":
        n, size = case["tokens"] * heads * dim, 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * n * size + 4 * case["tokens"], "flops": 3 * case["tokens"] * heads * case["rot"]}
    if case["op"] == "append":
        # the new keys and values in, the cache once more out, its values written
        size = 2 if case["dtype"] == "bf16" else 4
        live, slots = case["tokens"] - case["skipped"], case["pages"] * case["page"]
        return {"bytes": live * (2 * heads * dim * size + stored) + 8 * case["tokens"] + slots * (stored + 2 * heads * dim * 2),
                "flops": live * heads * (3 * case["rot"] + 2 * 5 * dim) + slots * heads * 2 * 2 * dim}
    q, kv = _whole(case["q"]), _whole(case["kv"])
    read = sum(n for c, n in zip(q, kv) if c)
    pairs = sum(sum(max(0, n - c + 1 + j) for j in range(c)) if case["causal"] else c * n for c, n in zip(q, kv))
    hq = heads * case["group"]
    return {"bytes": read * stored + 2 * 2 * sum(q) * hq * dim, "flops": 4 * dim * hq * pairs}


def _turned64(x, positions, freq, size, rot, layout):
    first, second = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    z = torch.polar(torch.full_like(freq, size).expand(len(positions), -1), torch.outer(positions.double(), freq))
    w = torch.complex(x[..., first], x[..., second]) * z[:, None]
    y = x.clone()
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _values64(data, scales, width):
    """The values of one array of packed rows [..., D / 2]."""
    groups = scales.shape[-2]
    byte = torch.arange(groups * GROUP // 2, device=data.device)
    out = torch.empty(*data.shape[:-1], groups * GROUP, dtype=torch.float64, device=data.device)
    for half in (0, 1):
        i = 2 * byte + half  # the code's place; its channel: block of `width`, then group, then lane
        channel = i // width % groups * GROUP + i // (width * groups) * width + i % width
        code = ((data >> (4 * half) & 15) ^ 8).double() - 8
        out[..., channel] = code * scales[..., channel // GROUP, 0].double() + scales[..., channel // GROUP, 1].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _turned64(s["x"].double(), s["positions"], s["freq"], s["size"], case["rot"], case["layout"])
    cache, page = s["cache"], case["page"]
    if case["op"] == "append":
        out = {n: _values64(cache[n], cache[n + "_scale"], w).transpose(1, 2).flatten(0, 1).contiguous() for n, w in (("k", 8), ("v", 4))}
        rows = s["written"]
        slots = s["slots"][rows].long()
        k = _turned64(s["k"].double(), s["positions"], s["freq"], s["size"], case["rot"], case["layout"])
        for name, x in (("k", k), ("v", s["v"].double())):
            g = x[rows].reshape(len(rows), case["heads"], -1, GROUP)
            step = ((g.max(-1).values - g.min(-1).values) / 15).float().bfloat16().double()  # held in bf16
            offset = (g.min(-1).values + 8 * step).float().bfloat16().double()
            code = torch.clip(torch.round((g - offset[..., None]) / step.clamp(min=1e-300)[..., None]), -8, 7)
            out[name][slots] = (code * step[..., None] + offset[..., None]).flatten(2)
        return out
    q, kv, group, dim = _whole(case["q"]), _whole(case["kv"]), case["group"], case["dim"]
    if sum(c * n for c, n in zip(q, kv)) * case["heads"] * group * dim > MOST64:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, (count, n) in enumerate(zip(q, kv)):
        if not count or not n:
            continue
        pages, start = s["table"][b, :-(-n // page)].long(), int(s["q_start"][b])
        for h in range(case["heads"]):
            k = _values64(cache["k"][pages, h], cache["k_scale"][pages, h], 8).flatten(0, 1)[:n]
            v = _values64(cache["v"][pages, h], cache["v_scale"][pages, h], 4).flatten(0, 1)[:n]
            rows = s["q"][start:start + count, h * group:(h + 1) * group].double()
            x = torch.einsum("cgd,nd->cgn", rows, k) / math.sqrt(dim)
            if case["causal"]:
                last = n - count + torch.arange(count, device="cuda")
                x = torch.where(torch.arange(n, device="cuda") <= last[:, None, None], x, -math.inf)
            out[start:start + count, h * group:(h + 1) * group] = torch.einsum(
                "cgn,nd->cgd", torch.softmax(x, -1).nan_to_num(0.0), v)
    return out
