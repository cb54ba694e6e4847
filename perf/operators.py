"""Decoding in 4 bits, as timed cases: the K/V cache that is quantised as it is written, attention over it, and the
linears with 4-bit weights.

Rows are held in groups of 64 channels: ``z`` is the least value of a group, ``s`` the spread over 15, both bf16, and a
channel is the code ``n`` (0 to 15, ties to even) of the value ``s n + z``.  A row of up to 64 channels is one group, a
longer one is padded to whole blocks of 128.  Codes are packed eight to a 32-bit word: channel ``i`` of the eight is
nibble ``i / 2`` (even) or ``4 + i / 2`` (odd), and in a block of 128 channels the words of its two groups alternate.
"""

import math

import torch

own = False

GROUP = 64


def listed():
    return [
        # one sequence decodes: its new token goes into the cache (1.3B configuration: 8 K/V heads of 128)
        dict(name="kv_token", kind="kv", B=1, T=1, hkv=8, D=128, page=128, late=True),
        # one step of a serving batch: 32 sequences at 32 different places of their caches
        dict(name="kv_tokens_32", kind="kv", B=32, T=1, hkv=8, D=128, page=128, late=True),
        # a second piece of a prompt behind a first one: heads of 64, pages of no round size, a ragged start
        dict(name="kv_piece_64", kind="kv", B=3, T=333, hkv=4, D=64, page=24, late=True),
        # eight whole prompts of the 1.3B configuration's length into empty caches
        dict(name="kv_prompts", kind="kv", B=8, T=4096, hkv=8, D=128, page=128, late=False),
        # a single user: one sequence of a few hundred rows
        dict(name="attn_one", kind="attn", B=1, rows=777, hq=16, hkv=8, D=128, page=128, window=0),
        # local layers of the Trinity recipe: three queries to a K/V head of 64, a sliding window, odd pages
        dict(name="attn_window_64", kind="attn", B=5, rows=1111, hq=12, hkv=4, D=64, page=24, window=256),
        # two long contexts, 8B configuration (4 queries to a K/V head)
        dict(name="attn_long", kind="attn", B=2, rows=32768, hq=32, hkv=8, D=128, page=128, window=0),
        # a serving batch of the 1.3B configuration, caches between 512 and 4096 rows
        dict(name="attn_batch", kind="attn", B=64, rows=4096, hq=16, hkv=8, D=128, page=128, window=0),
        # a single token through the output projection of the 1.3B configuration
        dict(name="linear_token", kind="linear", rows=1, N=2048, K=2048),
        # four tokens through gate and up of the 8B configuration
        dict(name="linear_wide", kind="linear", rows=4, N=28672, K=4096),
        # a serving batch through gate and up of the 1.3B configuration
        dict(name="linear_batch", kind="linear", rows=32, N=11264, K=2048),
        # a prompt of no round length through the down projection of the 1.3B configuration
        dict(name="linear_prompt", kind="linear", rows=777, N=2048, K=5632),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("kv", "attn", "attn", "linear", "linear"))
    page = rng.choice((16, 24, 64, 100, 128, 128, 256))
    if kind == "kv":
        hkv, D = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128))
        T = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        return dict(kind=kind, B=_log_int(rng, 1, max(1, min(64, 32768 // T))), T=T, hkv=hkv, D=D, page=page,
                    late=T == 1 or rng.random() < 0.5)
    if kind == "attn":
        hkv, D = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128))
        rows = _log_int(rng, 1, 65536)
        most = max(1, min(64, 64 * 4096 * 8 * 128 // (rows * hkv * D)))
        window = 0 if rng.random() < 0.7 else min(rows, _log_int(rng, 16, 2048))
        return dict(kind=kind, B=_log_int(rng, 1, most), rows=rows, hq=hkv * rng.choice((1, 2, 3, 4, 8)), hkv=hkv, D=D,
                    page=page, window=window)
    rows = _log_int(rng, 1, 64) if rng.random() < 0.8 else _log_int(rng, 65, 1024)
    N = _log_int(rng, 64, 16384)
    K = _log_int(rng, 64, 16384) if rng.random() < 0.4 else 64 * _log_int(rng, 1, 256)
    if rows > 64:
        N, K = min(N, 4096), min(K, 4096)
    return dict(kind=kind, rows=rows, N=N, K=K)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _width(channels):
    return 64 if channels <= 64 else (channels + 127) // 128 * 128


def _pages(c):
    rows = c["T"] + 1500 if c["kind"] == "kv" and c["late"] else c.get("T", c.get("rows"))
    return (rows + c["page"] - 1) // c["page"]


def _lengths(c):
    """Rows of each sequence's cache, longest first: an eighth of ``rows`` and up."""

    return [max(1, c["rows"] - b * c["rows"] * 7 // (8 * c["B"])) for b in range(c["B"])]


def _kv_rows(g, *shape):
    """Keys and values as projections leave them: channels of different width around different means."""

    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    width = torch.rand(shape[-1], generator=g, device="cuda").mul_(1.5).add_(0.25).to(torch.bfloat16)
    mean = torch.randn(shape[-1], generator=g, device="cuda").mul_(0.3).to(torch.bfloat16)
    return x.mul_(width).add_(mean)


def _kv_inputs(c, seed):
    g = _gen(seed)
    k = _kv_rows(g, c["B"], c["T"], c["hkv"], c["D"])
    v = _kv_rows(g, c["B"], c["T"], c["hkv"], c["D"])
    start = torch.randint(0, 1500, (c["B"],), generator=g, device="cuda", dtype=torch.int32) if c["late"] else None
    return k, v, start


def _attn_inputs(c, seed):
    g = _gen(seed)
    shape = (c["B"], _pages(c), c["hkv"], c["page"], c["D"])
    q = torch.randn(c["B"], c["hq"], c["D"], generator=g, device="cuda").to(torch.bfloat16)
    k, v = _quantized(_kv_rows(g, *shape)), _quantized(_kv_rows(g, *shape))
    order = torch.randperm(c["B"], generator=g, device="cuda")
    lengths = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)[order].contiguous()
    lo = (lengths - c["window"]).clamp_min(0) if c["window"] else None
    return q, k, v, lengths, lo


def _linear_inputs(c, seed):
    g = _gen(seed)
    x = torch.randn(c["rows"], c["K"], generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(c["N"], c["K"], generator=g, device="cuda").mul_(0.02).to(torch.bfloat16)
    return x, _quantized(w)


def prepare(case, seed):
    if case["kind"] == "kv":
        k, v, start = _kv_inputs(case, seed)
        rows = (case["B"], _pages(case), case["hkv"], case["page"])
        pools = [(torch.zeros(*rows, case["D"] // 2, dtype=torch.uint8, device="cuda"),
                  torch.zeros(*rows, case["D"] // GROUP, 2, dtype=torch.bfloat16, device="cuda")) for _ in range(2)]
        return dict(kind="kv", k=k, v=v, start=start, k_pool=pools[0], v_pool=pools[1])
    if case["kind"] == "attn":
        q, k, v, lengths, lo = _attn_inputs(case, seed)
        return dict(kind="attn", q=q, k_pool=k, v_pool=v, lengths=lengths, lo=lo)
    x, w = _linear_inputs(case, seed)
    return dict(kind="linear", x=x, w=w)


# ---- the plain form: elementary operations in 32 bits, codes in 64 ---------------------------------------------------
def _encode(x):
    """Codes, scales and least values of the groups of ``x [..., channels]``, padded to whole groups."""

    channels, width = x.shape[-1], _width(x.shape[-1])
    groups = torch.nn.functional.pad(x, (0, width - channels)).unflatten(-1, (-1, GROUP)).double()
    real = torch.arange(width, device=x.device).view(-1, GROUP) < channels
    z = groups.masked_fill(~real, math.inf).amin(-1, keepdim=True)
    top = groups.masked_fill(~real, -math.inf).amax(-1, keepdim=True)
    z, top = torch.where(real[:, :1], z, 0.0), torch.where(real[:, :1], top, 0.0)
    s = ((top - z) / 15.0).to(torch.bfloat16).double()
    n = torch.round((groups - z) / torch.where(s > 0, s, 1.0)).clamp(0, 15)
    n = torch.where(real & (s > 0), n, 0.0)
    return n.to(torch.uint8), torch.cat([s, z], dim=-1).to(torch.bfloat16)


def _pack(n):
    """``n [..., groups, 64]`` to bytes ``[..., groups * 32]``."""

    pair = 2 if n.shape[-2] > 1 else 1
    words = n.unflatten(-2, (-1, pair)).unflatten(-1, (8, 8)).transpose(-3, -2)          # [..., block, 8, pair, 8]
    low, high = words[..., [0, 4, 1, 5]], words[..., [2, 6, 3, 7]]
    return (low | (high << 4)).flatten(-4)


def _unpack(codes):
    """Bytes ``[..., groups * 32]`` to codes ``[..., groups, 64]``."""

    pair = 2 if codes.shape[-1] > 32 else 1
    b = codes.unflatten(-1, (-1, 8, pair, 4))
    low, high = b & 15, b >> 4
    n = torch.stack([low[..., 0], low[..., 2], high[..., 0], high[..., 2],
                     low[..., 1], low[..., 3], high[..., 1], high[..., 3]], dim=-1)
    return n.transpose(-3, -2).flatten(-2).flatten(-3, -2)


def _quantized(x):
    """What a program that keeps rows in 4 bits holds of them; a part at a time, so that it fits the card."""

    codes, affine = [], []
    for part in x.flatten(0, -2).split(max(1, (1 << 26) // x.shape[-1])):
        n, a = _encode(part)
        codes.append(_pack(n))
        affine.append(a)
    codes, affine = torch.cat(codes), torch.cat(affine)
    return codes.view(*x.shape[:-1], -1), affine.view(*x.shape[:-1], *affine.shape[1:])


def _values(codes, affine):
    """fp32 values ``[..., width]``."""

    a = affine.float()
    return (_unpack(codes).float() * a[..., :1] + a[..., 1:]).flatten(-2)


def _plain_kv(s):
    B, T, H, D = s["k"].shape
    page = s["k_pool"][0].shape[3]
    at = torch.arange(T, device="cuda")[None, :]
    at = at + s["start"][:, None].long() if s["start"] is not None else at.expand(B, T)
    b = torch.arange(B, device="cuda")[:, None].expand(B, T)
    out = []
    for x, (codes, affine) in ((s["k"], s["k_pool"]), (s["v"], s["v_pool"])):
        n, a = _encode(x)
        codes[b, at // page, :, at % page] = _pack(n)
        affine[b, at // page, :, at % page] = a
        out.append(_values(codes[b, at // page, :, at % page], affine[b, at // page, :, at % page]).to(x.dtype))
    return out


def _plain_attn(s):
    q = s["q"]
    B, hq, D = q.shape
    codes = s["k_pool"][0]
    hkv = codes.shape[2]
    k, v = (_values(*s[pool]).transpose(1, 2).flatten(2, 3) for pool in ("k_pool", "v_pool"))     # [B, hkv, rows, D]
    score = torch.matmul(q.float().view(B, hkv, hq // hkv, D), k.transpose(-1, -2)) * D ** -0.5
    at = torch.arange(k.shape[2], device="cuda")
    seen = at < s["lengths"][:, None]
    if s["lo"] is not None:
        seen = seen & (at >= s["lo"][:, None])
    score = torch.where(seen[:, None, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    return o.to(q.dtype).reshape(B, hq * D)


def _plain_linear(s):
    x = s["x"]
    w = _values(*s["w"])[:, :x.shape[1]]
    return torch.matmul(x.float(), w.t()).to(x.dtype)


def run(state):
    if own:
        from research_b200.ops import quantized as q4

        if state["kind"] == "kv":
            k_pool, v_pool = q4.Q4Rows(*state["k_pool"]), q4.Q4Rows(*state["v_pool"])
            q4.kv_write_paged_q4(state["k"], state["v"], k_pool, v_pool, state["start"])
            return list(q4.kv_read_paged_q4(k_pool, v_pool, state["k"].shape[1], state["start"]))
        if state["kind"] == "attn":
            return [q4.decode_attention_paged_q4(state["q"], q4.Q4Rows(*state["k_pool"]), q4.Q4Rows(*state["v_pool"]),
                                                 state["lengths"], state["lo"])]
        return [q4.linear_q4(state["x"], q4.Q4Rows(*state["w"]))]
    if state["kind"] == "kv":
        return _plain_kv(state)
    return [_plain_attn(state) if state["kind"] == "attn" else _plain_linear(state)]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "kv":
        rows = 2 * case["B"] * case["T"] * case["hkv"]
        held = case["D"] // 2 + case["D"] // 16
        return {"bytes": rows * (2 * case["D"] * 2 + 2 * held), "flops": 0}
    if case["kind"] == "attn":
        span = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
        held = case["D"] // 2 + case["D"] // 16
        return {"bytes": 2 * span * case["hkv"] * held + 2 * case["B"] * case["hq"] * case["D"] * 2,
                "flops": 4 * span * case["hq"] * case["D"]}
    width = _width(case["K"])
    return {"bytes": case["N"] * (width // 2 + width // 16) + 2 * case["rows"] * (case["K"] + case["N"]),
            "flops": 2 * case["rows"] * case["N"] * case["K"]}


# ---- the results in 64 bits, from the definition ---------------------------------------------------------------------
def _exact_rows(x):
    """The values that 16 levels leave of each group: the nearest level, the even one of two equally near."""

    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[-1], GROUP):
        part = x[..., first:first + GROUP].double()
        least = part.min(dim=-1, keepdim=True).values
        step = ((part.max(dim=-1, keepdim=True).values - least) / 15).to(torch.bfloat16).double()
        level = torch.zeros_like(part)
        for k in range(15):
            border = (k + 0.5) * step
            level += (part - least > border) | ((part - least == border) & (k % 2 == 1))
        out[..., first:first + GROUP] = torch.where(step > 0, level, 0.0) * step + least
    return out


def _exact_held(codes, affine, channels):
    """64-bit values of packed rows, a channel at a time."""

    width = codes.shape[-1] * 2
    out = torch.empty(*codes.shape[:-1], channels, dtype=torch.float64, device=codes.device)
    for c in range(channels):
        group, i = c // 64, c % 8
        word = c // 8 if width == 64 else c // 128 * 16 + c % 64 // 8 * 2 + group % 2
        nibble = i // 2 + 4 * (i % 2)
        n = (codes[..., word * 4 + nibble // 2] >> (4 * (nibble % 2))) & 15
        out[..., c] = n.double() * affine[..., group, 0].double() + affine[..., group, 1].double()
    return out


def exact(case, seed):
    if case["kind"] == "kv":
        k, v, _ = _kv_inputs(case, seed)
        return [_exact_rows(k), _exact_rows(v)]
    if case["kind"] == "attn":
        q, k_held, v_held, lengths, lo = _attn_inputs(case, seed)
        group = case["hq"] // case["hkv"]
        out = torch.zeros(case["B"], case["hq"], case["D"], dtype=torch.float64, device="cuda")
        for b in range(case["B"]):
            first, last = 0 if lo is None else int(lo[b]), int(lengths[b])
            k, v = (_exact_held(codes[b], affine[b], case["D"]).permute(0, 2, 1, 3).reshape(-1, case["hkv"], case["D"])
                    for codes, affine in (k_held, v_held))
            for h in range(case["hq"]):
                weight = torch.softmax(k[first:last, h // group] @ q[b, h].double() / math.sqrt(case["D"]), dim=0)
                out[b, h] = weight @ v[first:last, h // group]
        return [out.view(case["B"], -1)]
    x, (codes, affine) = _linear_inputs(case, seed)
    return [x.double() @ _exact_held(codes, affine, case["K"]).t()]
