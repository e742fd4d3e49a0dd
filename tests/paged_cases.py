"""Paged batches with a 64-bit reference, for the windowed and the 4-bit paths.

A batch draws the K and V rows of every cached token, deals a permutation of the
pool's blocks to the sequences, and appends the rows through the pool's own
append (slots that nothing writes hold NaN patterns).  `held` gives the values
that the pool's codec leaves of a row, from the codec's definition, in 64 bits;
`attend` is the masked softmax attention over them, in 64 bits, on the CPU, with
the sum of p * |v| beside each output, which rounded probabilities are off by a
share of.

Tolerance of an output with reference r, A = sum p |v| and F (below):
    u * |r| + c * A + 2^-25 * F
u: half a step of the io type (bf16 2^-8, fp16 2^-11), taken 1% larger for the
second-order term.  c: probabilities enter the P V product as a pair hi + lo (bf16
pages 2^-16, FP8 pages 2^-22) or, on f16 pages and in the decode of 4-bit ones, as one f16 (2^-11); the
f32 score of up to 128 products of about 2^5 in magnitude (128 * 2^-24 * 2^5 * ln 2
relative in p: 2^-12.5 at the very worst, rounding errors of both signs and far
fewer than 128 of them at that size: 2^-14) and ex2.approx (2^-22) add to it.  So
c = 2^-13 covers hi + lo, 2^-11 + 2^-13 one f16.
F, for f16, FP8 and 4-bit pages: f16 values below 2^-14 have a fixed step of 2^-24, so a small probability that
enters the product as f16 (the lo half of a pair, or the one f16) is off by up to 2^-25 whatever its size.  The
unnormalised e = exp(s - m), m at most the largest score, enters it (FP8 pages: e times the row's V scale t), against
the held value v (FP8: v / t), and is divided by sum e >= sum exp(s - max): F = sum_j |v_j| / t_j / sum_j exp(s_j - max),
over the visible keys.
"""
import math

import numpy as np
import torch

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
PAGE = 16
HIDDEN = -1            # as a block id: 0xFFFFFFFF


def nearest(x, bits, low, most):
    """x (64 bits) to the nearest value of `bits` significant bits, exponents from `low`, at most `most`; ties to even."""
    e = torch.frexp(x.abs())[1] - 1
    step = torch.ldexp(torch.ones_like(x), e.clamp(min=low) - (bits - 1))
    return (torch.round(x / step) * step).clamp(-most, most)


def held(x, kv):
    """What the pool keeps of io rows [..., D], in 64 bits."""
    x = x.double()
    if kv in ("f16", "bf16"):
        return x
    if kv == "fp8":        # "ocp": one f32 scale per row, quotients in f32, E4M3 to nearest even
        s = (x.abs().amax(-1, keepdim=True) / 448.0).float().double()
        s[s == 0] = 1.0
        return nearest((x / s).float().double(), 4, -6, 448.0) * s
    # (magnitudes past 6 * 448 saturate alike: cut off before infinities meet frexp)
    g = x.clamp(-1e6, 1e6).unflatten(-1, (-1, 16))      # "fp4": an E4M3 scale per 16 elements, E2M1 codes
    s = nearest(g.abs().amax(-1, keepdim=True) / 6.0, 4, -6, 448.0)
    return (nearest(g / s.masked_fill(s == 0, math.inf), 2, 0, 6.0) * s).flatten(-2)


def attend(q, k, v, pos, window=0, sinks=0, causal=True, scale=None, v_scale=None):
    """q [n][Hq][D] at positions pos [n]; k, v [S][Hkv][D] (64 bits) -> outputs, A, F (v_scale: FP8 pages' t [S][Hkv])."""
    n, Hq, D = q.shape
    S, Hkv, _ = k.shape
    q, g = q.double(), Hq // Hkv
    j = torch.arange(S)[None, :]
    seen = (j <= pos[:, None]) if causal else torch.ones(n, S, dtype=torch.bool)
    if window:
        seen &= (pos[:, None] - j < window) | (j < sinks)
    k = k.repeat_interleave(g, 1)
    v = torch.where(seen.any(0)[:, None, None], v, torch.zeros_like(v)).repeat_interleave(g, 1)
    s = torch.einsum("nhd,shd->nhs", q, k) * (1.0 / math.sqrt(D) if scale is None else scale)
    s = torch.where(seen[:, None, :], s, torch.full_like(s, -math.inf))
    p = torch.softmax(s, -1)
    t = torch.ones(S, Hkv, dtype=torch.float64) if v_scale is None else v_scale
    mass = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1, keepdim=True)
    F = torch.einsum("ns,shd->nhd", seen.double(), v.abs() / t.repeat_interleave(g, 1)[..., None]) / mass
    return torch.einsum("nhs,shd->nhd", p, v), torch.einsum("nhs,shd->nhd", p, v.abs()), F


def v_scales(v, kv):
    """t of attend: the f32 scale of FP8 rows."""
    if kv != "fp8":
        return None
    s = (v.double().abs().amax(-1) / 448.0).float().double()
    s[s == 0] = 1.0
    return s


def check(got, ref, A, F, io, kv, what=""):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    u = torch.finfo(TYPES[io]).eps / 2 * 1.01
    c = 2.0 ** -13 + (2.0 ** -11 if kv in ("f16", "fp4") else 0.0)
    tol = u * ref.abs() + c * A + (0.0 if kv == "bf16" else 2.0 ** -25 * F) + 2.0 ** -25
    worst = ((got - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3g} times the tolerance"


class Batch:
    """totals[b] tokens per sequence in one pool (num_layers layers, the same rows in each)."""

    def __init__(self, seed, kv, io, D, Hq, Hkv, totals, layers=1, dev=0, spare=5, stride_extra=2, scale=1.0,
                 max_batch=None, fp8_mode="ocp"):
        from voidweb_b200.kv import KvPool, PoolSpec
        self.kv, self.io, self.D, self.Hq, self.Hkv, self.totals = kv, io, D, Hq, Hkv, list(totals)
        self.g = torch.Generator().manual_seed(seed)
        self.dt, self.dev, self.layers = TYPES[io], torch.device("cuda", dev), layers
        B, pages = len(totals), [(t + 15) // 16 for t in totals]
        self.B, self.nb = B, sum(pages) + spare
        perm = torch.randperm(self.nb, generator=self.g)
        self.table = torch.full((B, max(pages) + stride_extra), HIDDEN, dtype=torch.int64)
        at = 0
        for b, n in enumerate(pages):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.k = [self.rows(t, Hkv, scale) for t in totals]
        self.v = [self.rows(t, Hkv, scale) for t in totals]
        self.pool = KvPool(PoolSpec(num_layers=layers, num_kv_heads=Hkv, head_dim=D, num_blocks=self.nb, kv_dtype=kv,
                                    io_dtype=io, fp8_mode=fp8_mode, max_batch=max_batch or max(B, 1)), device=dev)
        self.pool.pages_u8().fill_(0xFF)
        if kv == "fp8":
            self.pool.scales_f32().fill_(math.nan)

    def rows(self, n, H, scale=1.0):
        return (torch.randn(n, H, self.D, generator=self.g) * scale).to(self.dt)

    def slots(self, b, first=0, last=None):
        p = torch.arange(first, self.totals[b] if last is None else last)
        return self.table[b, p // PAGE] * PAGE + p % PAGE

    def fill(self, keep=None):
        """Append tokens [0, keep[b]) of every sequence (all of them by default) in every layer."""
        keep = self.totals if keep is None else keep
        s = torch.cat([self.slots(b, 0, n) for b, n in enumerate(keep)])
        k = torch.cat([x[:n] for x, n in zip(self.k, keep)])
        v = torch.cat([x[:n] for x, n in zip(self.v, keep)])
        if len(s):
            for l in range(self.layers):
                self.pool.append(l, k.to(self.dev), v.to(self.dev), s.to(self.dev))
        return self

    def overwrite(self, b, first, last, value):
        """Rows [first, last) of sequence b become `value` in every element."""
        if last <= first:
            return
        r = torch.full((last - first, self.Hkv, self.D), value, dtype=self.dt, device=self.dev)
        for l in range(self.layers):
            self.pool.append(l, r, r, self.slots(b, first, last).to(self.dev))

    def device_table(self, hide=None):
        """The block tables on the device; hide(b, page) -> the entry is 0xFFFFFFFF instead."""
        t = self.table.clone()
        if hide is not None:
            for b in range(self.B):
                for pg in range(t.shape[1]):
                    if hide(b, pg):
                        t[b, pg] = HIDDEN
        return t.to(torch.int32).to(self.dev)

    def lens(self, lens=None):
        return torch.tensor(self.totals if lens is None else lens, dtype=torch.int32, device=self.dev)


def hidden_pages(total_first, total_last, window, sinks):
    """Pages that no query at positions total_first .. total_last sees (a function of the page)."""
    lo = max(0, total_first - window + 1)
    return lambda pg: pg * PAGE >= sinks and (pg + 1) * PAGE <= lo
