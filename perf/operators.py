"""The 4-bit KV cache and windowed attention: what is timed and compared, and its plain forms.

Operators, all on one layer of a paged pool:

  store           rows of a prompt's K and V are quantised into a 4-bit pool and read back as
                  io-typed values (a cache handed over between workers)
  fp4_decode      one query token per sequence over a 4-bit pool, optionally windowed
  fp4_prefill     chunks of query tokens over a 4-bit pool, causal, optionally windowed
  window_decode   one query token per sequence, a sliding window and a few first tokens
                  (sinks), over f16 / bf16 / FP8 pools
  window_prefill  chunks of query tokens under the same mask, over f16 / bf16 / FP8 pools

A 4-bit row: every 16 consecutive elements share the scale s = E4M3(amax / 6), an element x is
held as E2M1(x / s) (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; both roundings to nearest,
ties to the even code), and stands for code * s; a group whose scale rounds to 0 is held as 0.

The mask: the token at position p sees the keys j <= p with p - j < window or j < sinks.
"""
import math
import random
import zlib

import torch

own = False

PAGE = 16
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a page and a token of a small model's cache: launch latency
        dict(name="store-17", op="store", io="f16", Hq=14, Hkv=2, D=64, B=1, lo=17, hi=17),
        # a long prompt of an 8-billion-parameter model handed over to a 4-bit pool
        dict(name="store-8191", op="store", io="bf16", Hq=32, Hkv=8, D=128, B=1, lo=8191, hi=8191),
        # one user, a short chat, 64-element heads
        dict(name="fp4-decode-1", op="fp4_decode", io="f16", kv="fp4", Hq=14, Hkv=2, D=64, B=1, lo=193, hi=193,
             window=0, sinks=0),
        # a serving batch of Qwen2.5-7B
        dict(name="fp4-decode-qwen-16", op="fp4_decode", io="bf16", kv="fp4", Hq=28, Hkv=4, D=128, B=16, lo=512,
             hi=4096, window=0, sinks=0),
        # a large batch of Llama-3-8B with long contexts: bandwidth
        dict(name="fp4-decode-llama-64", op="fp4_decode", io="bf16", kv="fp4", Hq=32, Hkv=8, D=128, B=64, lo=1024,
             hi=16384, window=0, sinks=0),
        # chunks of four prompts of Qwen2.5-7B after a cached prefix
        dict(name="fp4-prefill-qwen-4", op="fp4_prefill", io="bf16", kv="fp4", Hq=28, Hkv=4, D=128, B=4, lo=0, hi=2048,
             nlo=2048, nhi=2048, window=0, sinks=0),
        # short questions over cached documents
        dict(name="fp4-prefill-short", op="fp4_prefill", io="f16", kv="fp4", Hq=32, Hkv=8, D=128, B=7, lo=100, hi=1500,
             nlo=1, nhi=77, window=0, sinks=0),
        # one user far beyond the window: latency
        dict(name="window-decode-1", op="window_decode", io="bf16", kv="bf16", Hq=28, Hkv=4, D=128, B=1, lo=20011,
             hi=20011, window=1000, sinks=4),
        # the serving batch with long contexts
        dict(name="window-decode-qwen-16", op="window_decode", io="bf16", kv="bf16", Hq=28, Hkv=4, D=128, B=16,
             lo=2048, hi=32768, window=4096, sinks=4),
        # the large batch over FP8 pages
        dict(name="window-decode-llama-64", op="window_decode", io="bf16", kv="fp8", Hq=32, Hkv=8, D=128, B=64,
             lo=1024, hi=32768, window=4096, sinks=16),
        # chunks of long prompts behind the window
        dict(name="window-prefill-qwen-4", op="window_prefill", io="bf16", kv="bf16", Hq=28, Hkv=4, D=128, B=4, lo=0,
             hi=8192, nlo=2048, nhi=2048, window=1024, sinks=4),
        # ragged short chunks of a small model
        dict(name="window-prefill-ragged", op="window_prefill", io="f16", kv="f16", Hq=14, Hkv=2, D=64, B=9, lo=0,
             hi=700, nlo=1, nhi=200, window=99, sinks=5),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    while True:
        op = rng.choice(("store", "fp4_decode", "fp4_prefill", "window_decode", "window_prefill"))
        io = rng.choice(("f16", "bf16"))
        D = rng.choice((64, 128))
        Hkv = rng.choice((1, 2, 4, 8))
        c = dict(op=op, io=io, Hq=Hkv * spread(1, 16), Hkv=Hkv, D=D)
        if op == "store":
            n = spread(1, 8191)
            return dict(c, B=1, lo=n, hi=n)
        if op.startswith("fp4"):
            kv = "fp4"
            windowed = rng.random() < 0.4
        else:
            kv = rng.choice((io, "fp8")) if D == 128 else io
            windowed = True
        c.update(kv=kv, window=spread(1, 4096) if windowed else 0, sinks=rng.choice((0, 1, 4, spread(1, 64))) if windowed else 0)
        if op.endswith("decode"):
            hi = spread(1, 32768 if windowed else 16384)
            c.update(B=spread(1, 64), lo=spread(1, hi), hi=hi)
            if work(c)["bytes"] <= 4.4e8:
                return c
        else:
            hi = spread(1, 8192) - 1
            nhi = spread(1, 2048)
            c.update(B=spread(1, 9), lo=rng.randint(0, hi), hi=hi, nlo=spread(1, nhi), nhi=nhi)
            if c["B"] * c["Hq"] * nhi * (hi + nhi) <= 4 * 28 * 2048 * (8192 + 2048) and work(c)["flops"] <= 1.3e11:
                return c


def _lens(case):
    """Cached lengths: from the case alone, spread over its range."""
    rng = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    lo, hi, B = case["lo"], case["hi"], case["B"]
    lens = [int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1 for _ in range(B)]
    return [min(hi, max(lo, n)) for n in lens]


def _chunks(case):
    """Query tokens of each sequence's chunk: from the case alone."""
    rng = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()) + 1)
    return [rng.randint(case["nlo"], case["nhi"]) for _ in range(case["B"])]


def _visible(p, window, sinks):
    """Keys that the token at position p sees."""
    return p + 1 if not window or p + 1 <= window else window + min(sinks, p + 1 - window)


def _pairs(case):
    """(query token, key) pairs of a prefill under its mask."""
    return sum(_visible(c + i, case["window"], case["sinks"]) for c, n in zip(_lens(case), _chunks(case)) for i in range(n))


def _row_bytes(case):
    D = case["D"]
    return {"fp4": D // 2 + D // 16, "fp8": D + 4}.get(case.get("kv", "fp4"), 2 * D)


def work(case):
    Hq, Hkv, D, B = case["Hq"], case["Hkv"], case["D"], case["B"]
    lens = _lens(case)
    if case["op"] == "store":
        n = lens[0]
        # rows in, codes and scales out, codes and scales in, rows out; a division and a product for each element
        return {"bytes": 2 * n * Hkv * (2 * 2 * D + 2 * _row_bytes(case)) + 8 * n, "flops": 4 * n * Hkv * D}
    w, s = case["window"], case["sinks"]
    if case["op"].endswith("decode"):
        keys = sum(_visible(n - 1, w, s) for n in lens)
        pages = sum((_visible(n - 1, w, s) + PAGE - 1) // PAGE for n in lens)
        return {"bytes": 2 * keys * Hkv * _row_bytes(case) + 2 * B * Hq * D * 2 + 4 * pages + 4 * B,
                "flops": 4 * keys * Hq * D}
    ns = _chunks(case)
    keys = 0
    for c, n in zip(lens, ns):
        first = max(0, c - w + 1) if w else 0
        keys += c + n - max(0, first - s)
    return {"bytes": 2 * keys * Hkv * _row_bytes(case) + 2 * sum(ns) * Hq * D * 2 + 4 * (keys // PAGE) + 8 * B,
            "flops": 4 * _pairs(case) * Hq * D}


def _rows(shape, gen, dtype, spread):
    """Normal values; `spread` (K): a few channels are several times as large as the others, as a model's keys are."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if spread:
        g = torch.randn(shape[-1], generator=gen, device="cuda", dtype=torch.float32)
        x *= torch.exp(0.5 * g)
    return x.to(dtype)


def _inputs(case, seed):
    """K and V rows of every cached token (sequence after sequence), the pages they lie in, and the queries."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, Hq, Hkv, D, B = TYPES[case["io"]], case["Hq"], case["Hkv"], case["D"], case["B"]
    lens = _lens(case)
    ns = _chunks(case) if case["op"].endswith("prefill") else [0] * B
    totals = [a + b for a, b in zip(lens, ns)]
    pages = [(t + PAGE - 1) // PAGE for t in totals]
    nb = sum(pages) + 16
    perm = torch.randperm(nb, generator=gen, device="cuda")
    table = torch.zeros(B, max(pages) + 1, dtype=torch.int64, device="cuda")
    start = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[start:start + n]
        start += n
    T = sum(totals)
    owner = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(totals, device="cuda"), output_size=T)
    first = torch.tensor([0] + totals, device="cuda").cumsum(0)
    pos = torch.arange(T, device="cuda") - first[owner]
    slots = table[owner, pos // PAGE] * PAGE + pos % PAGE
    k, v = _rows((T, Hkv, D), gen, dt, True), _rows((T, Hkv, D), gen, dt, False)
    rows = sum(ns) if case["op"].endswith("prefill") else B
    q = _rows((rows, Hq, D), gen, dt, False)
    return dict(k=k, v=v, q=q, table=table, slots=slots, nb=nb, lens=lens, ns=ns, totals=totals)


def _quantise(x):
    """Codes (two to a byte, the even element in the low half) and scales of rows, in 32 bits: every border that decides
    is a product of few bits, so the quotients of 32 bits fall on the right side of it."""
    g = x.float().unflatten(-1, (-1, 16))
    # (by a tensor: a division by a number would be a product with its rounded inverse)
    s = (g.abs().amax(-1) / torch.tensor(6.0, device="cuda")).clamp(max=448.0).to(torch.float8_e4m3fn)
    f = s.float().unsqueeze(-1)
    a = torch.where(f > 0, g.abs() / f, torch.zeros_like(g))
    c = (a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()
    c = c + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
    c = (c + 8 * torch.signbit(g).byte()).flatten(-2)
    return c[..., 0::2] + 16 * c[..., 1::2], s


def _values(codes, s):
    """What codes and scales stand for, in 32 bits."""
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    return (table[c].unflatten(-1, (-1, 16)) * s.float().unsqueeze(-1)).flatten(-2)


def _pool_of(case, i):
    from voidweb_b200.kv import KvPool, PoolSpec
    kv = case.get("kv", "fp4")
    pool = KvPool(PoolSpec(num_layers=1, num_kv_heads=case["Hkv"], head_dim=case["D"], num_blocks=i["nb"], kv_dtype=kv,
                           io_dtype=case["io"], fp8_mode="ocp", max_batch=64))
    pool.pages_u8().fill_(0xFF)      # NaN patterns in every slot that nothing writes
    if kv == "fp8":
        pool.scales_f32().fill_(math.nan)
    return pool


def prepare(case, seed):
    i = _inputs(case, seed)
    st = dict(case=case, q=i["q"], lens=torch.tensor(i["lens"], dtype=torch.int32, device="cuda"))
    kv = case.get("kv", "fp4")
    if case["op"] == "store":
        st.update(k=i["k"], v=i["v"], slots=i["slots"], nb=i["nb"])
    if case["op"].endswith("prefill"):
        st["cu"] = torch.tensor([0] + i["ns"], device="cuda").cumsum(0).int()
        st["chunk"], st["longest"] = max(i["ns"]), max(i["totals"])
    st["table"] = i["table"].int()
    if own:
        st["pool"] = _pool_of(case, i)
        st["out"] = torch.empty_like(i["q"])
        if case["op"] != "store":
            st["pool"].append(0, i["k"], i["v"], i["slots"])
        return st
    if case["op"] != "store":
        def paged(x):
            out = torch.zeros((i["nb"] * PAGE,) + x.shape[1:], dtype=x.dtype, device="cuda")
            out.view(torch.uint8)[i["slots"]] = x.contiguous().view(torch.uint8)
            return out
        for n in ("k", "v"):
            if kv == "fp4":
                codes, s = _quantise(i[n])
                st[n] = (paged(codes), paged(s))
            elif kv == "fp8":
                s = i[n].float().abs().amax(-1) / torch.tensor(448.0, device="cuda")
                s = torch.where(s == 0, torch.ones_like(s), s)
                st[n] = (paged((i[n].float() / s.unsqueeze(-1)).to(torch.float8_e4m3fn)), paged(s.unsqueeze(-1)))
            else:
                st[n] = (paged(i[n]), None)
        st["seen"] = int(min(max(i["totals"]), case["window"] + case["sinks"])) if case["window"] else int(max(i["totals"]))
    return st


def run(state):
    case = state["case"]
    if own:
        pool, out = state["pool"], state["out"]
        if case["op"] == "store":
            pool.append(0, state["k"], state["v"], state["slots"])
            return list(pool.gather(0, state["table"][0], case["hi"])[:2])
        if case["op"].endswith("decode"):
            return pool.paged_decode(0, state["q"], state["table"], state["lens"], out, window=case["window"],
                                     sinks=case["sinks"])
        return pool.paged_prefill(0, state["q"], state["cu"], state["lens"], state["table"], out,
                                  window=case["window"], sinks=case["sinks"])
    if case["op"] == "store":
        return _store(state)
    return (_decode if case["op"].endswith("decode") else _prefill)(state)


def _store(st):
    out = []
    for x in (st["k"], st["v"]):
        codes, s = _quantise(x)
        c = torch.zeros((st["nb"] * PAGE,) + codes.shape[1:], dtype=torch.uint8, device="cuda")
        f = torch.zeros((st["nb"] * PAGE,) + s.shape[1:], dtype=torch.uint8, device="cuda")
        c[st["slots"]], f[st["slots"]] = codes, s.view(torch.uint8)
        n = torch.arange(len(x), device="cuda")
        slots = st["table"][0].long()[n // PAGE] * PAGE + n % PAGE
        out.append(_values(c[slots], f[slots].view(torch.float8_e4m3fn)).to(x.dtype).transpose(0, 1).contiguous())
    return out


def _cached(kv, slots, kind):
    """The rows in `slots`, in 32 bits."""
    x, s = kv
    if kind == "fp4":
        return _values(x[slots], s.view(torch.uint8)[slots].view(torch.float8_e4m3fn))
    if kind == "fp8":
        return x.view(torch.uint8)[slots].view(torch.float8_e4m3fn).float() * s[slots]
    return x[slots].float()


def _softmax(s, mask):
    s = s.masked_fill(~mask, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _decode(st):
    c, L = st["case"], st["lens"].long().unsqueeze(1)
    n = torch.arange(st["seen"], device="cuda").unsqueeze(0)
    pos = n
    if c["window"]:      # the first tokens, then the window
        low = (L - c["window"]).clamp(min=c["sinks"])
        pos = torch.where(n < c["sinks"], n, low + n - c["sinks"])
    mask = pos < L
    pos = torch.minimum(pos, L - 1)
    slots = torch.gather(st["table"].long(), 1, pos // PAGE) * PAGE + pos % PAGE
    q = st["q"].float().unflatten(1, (c["Hkv"], -1))
    s = torch.matmul(q, _cached(st["k"], slots, c["kv"]).permute(0, 2, 3, 1)) / math.sqrt(c["D"])
    p = _softmax(s, mask[:, None, None, :])
    return torch.matmul(p, _cached(st["v"], slots, c["kv"]).transpose(1, 2)).flatten(1, 2).to(st["q"].dtype)


def _prefill(st):
    c, cu, start = st["case"], st["cu"].long(), st["lens"].long()
    i = torch.arange(st["chunk"], device="cuda").unsqueeze(0)
    row = cu[:-1, None] + i
    live = row < cu[1:, None]
    row = torch.where(live, row, torch.zeros_like(row))
    p = (start[:, None] + i)[:, :, None]
    j = torch.arange(st["longest"], device="cuda")[None, None, :]
    mask = j <= p
    if c["window"]:
        mask = mask & ((p - j < c["window"]) | (j < c["sinks"]))
    key = torch.minimum(j[:, 0], (start + cu[1:] - cu[:-1])[:, None] - 1)
    slots = torch.gather(st["table"].long(), 1, key // PAGE) * PAGE + key % PAGE
    q = st["q"][row].float().unflatten(2, (c["Hkv"], -1)).permute(0, 2, 3, 1, 4)       # [B][Hkv][g][n][D]
    k = _cached(st["k"], slots, c["kv"]).permute(0, 2, 3, 1).unsqueeze(2)
    v = _cached(st["v"], slots, c["kv"]).transpose(1, 2).unsqueeze(2)
    w = _softmax(torch.matmul(q, k) / math.sqrt(c["D"]), mask[:, None, None])
    o = torch.matmul(w, v).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[live].to(st["q"].dtype)


def exact(case, seed):
    """The definition in 64 bits, one sequence and one KV head at a time."""
    i = _inputs(case, seed)
    kv = case.get("kv", "fp4")

    def held(x):
        x = x.double()
        if kv in ("f16", "bf16"):
            return x
        if kv == "fp8":
            # an FP8 row's scale and its elements' quotients are defined as values of 32 bits
            s = (x.abs().amax(-1, keepdim=True) / 448.0).float().double()
            s[s == 0] = 1.0
            return _nearest((x / s).float().double(), 4, -6, 448.0) * s
        g = x.reshape(x.shape[:-1] + (-1, 16))
        s = _nearest(g.abs().amax(-1, keepdim=True) / 6.0, 4, -6, 448.0)
        return (_nearest(g / s.masked_fill(s == 0, math.inf), 2, 0, 6.0) * s).reshape(x.shape)

    if case["op"] == "store":
        return [held(i["k"]).transpose(0, 1).contiguous(), held(i["v"]).transpose(0, 1).contiguous()]
    group, outs, at, row = case["Hq"] // case["Hkv"], [], 0, 0
    for b in range(case["B"]):
        total = i["totals"][b]
        n = i["ns"][b] or 1
        k, v = held(i["k"][at:at + total]), held(i["v"][at:at + total])
        q = i["q"][row:row + n].double()
        at, row = at + total, row + n
        p = torch.arange(total - n, total, device="cuda")[:, None]
        j = torch.arange(total, device="cuda")[None, :]
        seen = (j <= p) & ((j > p - case["window"]) | (j < case["sinks"])) if case["window"] else j <= p
        o = torch.empty_like(q)
        for h in range(case["Hkv"]):
            for m in range(h * group, (h + 1) * group):
                s = q[:, m] @ k[:, h].T / case["D"] ** 0.5
                s = torch.where(seen, s, torch.full_like(s, -math.inf))
                o[:, m] = torch.softmax(s, -1) @ v[:, h]
        outs.append(o)
    return torch.cat(outs)


def _nearest(x, bits, low, most):
    """x to the nearest value of `bits` significant bits, exponents from `low` on, at most `most`; ties to the even one."""
    e = torch.frexp(x.abs())[1].to(torch.int32) - 1
    step = torch.ldexp(torch.ones_like(x), e.clamp(min=low) - (bits - 1))
    return (torch.round(x / step) * step).clamp(-most, most)
