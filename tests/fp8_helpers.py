"""A cache in 8 bits and attention over it, restated in 64 bits: what the kernels are compared with."""

from __future__ import annotations

import math

import torch

EMAX = 60


def two_to(e: torch.Tensor) -> torch.Tensor:
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest number of e4m3 (ties to the even step) of float64 numbers up to 448: steps of 2^-9 below 2^-6, eight to an octave above."""
    m, e = torch.frexp(y.abs())  # |y| = m 2^e, m in [1/2, 1)
    step = two_to(torch.where(y == 0, torch.full_like(e, -6), e - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def hold(x: torch.Tensor) -> "tuple[torch.Tensor, torch.Tensor]":
    """(values that rows x [..., d] are kept as, scale bytes), from the format's definition."""
    x = x.double()
    top = x.abs().amax(-1)
    bad = ~(x.abs() <= 448 * 2.0 ** EMAX).all(-1)
    top = torch.where(bad, torch.ones_like(top), top)
    e = torch.full(top.shape, -EMAX, dtype=torch.int64, device=x.device)
    for k in range(-EMAX, EMAX):  # one step up wherever the row does not fit yet
        e = torch.where((e == k) & (top > 448 * 2.0 ** k), e + 1, e)
    s = two_to(e)[..., None]
    values = torch.where(bad[..., None], torch.full_like(x, math.nan), e4m3(torch.where(bad[..., None], torch.zeros_like(x), x) / s) * s)
    return values, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


class Case:
    """A paged cache of ``held[r]`` keys per request plus the step's own ``n[r]``, in pages scattered over a pool that holds more."""

    def __init__(self, n, held, Hq, Hkv, dh, page, seed=0, bits8=True, device="cuda", spread=1.0):
        gen = torch.Generator().manual_seed(seed)
        self.n, self.held, self.Hq, self.Hkv, self.dh, self.page = list(n), list(held), Hq, Hkv, dh, page
        R, self.N = len(n), sum(n)
        per = [-(-(a + b) // page) for a, b in zip(n, held)]
        self.P = sum(per) + 3
        order = torch.randperm(self.P, generator=gen).tolist()
        self.table = torch.full((R, max(per) + 1), -1, dtype=torch.int32)
        for r, p in enumerate(per):
            self.table[r, :p] = torch.tensor([order.pop() for _ in range(p)], dtype=torch.int32)
        self.req = torch.repeat_interleave(torch.arange(R), torch.tensor(n)).to(torch.int32)
        firsts = [sum(n[:r]) for r in range(R + 1)]
        self.cu_q, self.q_start = torch.tensor(firsts, dtype=torch.int32), torch.tensor(held, dtype=torch.int32)
        self.places = torch.tensor([held[r] + j for r in range(R) for j in range(n[r])], dtype=torch.int32)
        self.positions = self.places.clone()
        self.rows = torch.randn((self.P, 2, Hkv, page, dh), generator=gen).to(torch.bfloat16).double()
        self.rows *= torch.exp2(torch.round(spread * torch.randn((self.P, 2, Hkv, page, 1), generator=gen))).double()
        if bits8:
            self.rows, scales = hold(self.rows)
            self.set_rows8(scales)
        else:
            self.pages, self.scales = self.rows.to(torch.bfloat16), None
        self.q = (1.5 * torch.randn((self.N, Hq, dh), generator=gen)).to(torch.bfloat16)
        self.bits8, self.device, self.masks = bits8, device, None
        self.weights = 2.0 ** -11 if bits8 else 2.0 ** -8  # rounding of the weights; served() says otherwise
        self.status = torch.zeros(1, dtype=torch.int32)
        self.scale = dh ** -0.5

    def set_rows8(self, scales):
        self.scales = scales
        s = two_to(scales.long().clamp(max=200) - 127)[..., None]
        self.pages = torch.nan_to_num(self.rows / s, nan=0.0).to(torch.float32).to(torch.float8_e4m3fn)

    def tree(self, seed=1, parents=None):
        from jax_llm_examples_b200.kernels import api as K

        gen = torch.Generator().manual_seed(seed)
        words = -(-max(self.n) // 32)
        self.masks = torch.zeros((self.N, words), dtype=torch.int32)
        at = 0
        for r, m in enumerate(self.n):
            p = parents[r] if parents else [int(torch.randint(-1, j, (1,), generator=gen)) if j else -1 for j in range(m)]
            depth, bits = K.tree_masks(p)
            for j in range(m):
                self.positions[at + j] = self.held[r] + depth[j]
                self.masks[at + j, :len(bits[j])] = torch.tensor(bits[j], dtype=torch.int32)
            at += m
        return self

    def to_device(self):
        for k, v in list(vars(self).items()):
            if isinstance(v, torch.Tensor) and k != "rows":
                setattr(self, k, v.to(self.device))
        return self

    def served(self, max_count):
        """To be called for the items that a kernel gets: the tcgen05 form rounds its weights to bfloat16 over either cache."""
        from jax_llm_examples_b200.kernels import api as K

        form = K.attention_rows_form(max_count * (self.Hq // self.Hkv), self.page, True)
        self.weights = 2.0 ** -11 if self.bits8 and form != "attention_rows_tc" else 2.0 ** -8

    def items(self, cut, which=lambda n: True):
        """(int32 [n, 2], count, largest count)"""
        t = [(int(self.cu_q[r]) + o, min(cut, m - o)) for r, m in enumerate(self.n) if which(m) for o in range(0, m, cut)]
        return torch.tensor(t, dtype=torch.int32, device=self.device), len(t), max(c for _, c in t)

    def want(self, chunk=0, window=0, temper=0.0, floor=1.0, sink=None, slopes=None, cap=0.0):
        """(output, how far a kernel's may be) in float64 on the CPU, [N, Hq, dh].

        The bound, element by element: half a step of the bfloat16 output (2^-8 of it); and of A = sum_j w_j |v_j|: the weights'
        rounding for the product (2^-11 in float16, 2^-8 in bfloat16), twice the scores' error (numerator and sum): the order of
        a 32-bit sum of dh products, 2 dh 2^-24 of the largest sum of |q k|, and 2^-18 for the exponent's argument and the
        exponential.  Weights below 2^-14 of the largest are off by 2^-25 in float16 whatever their size: a last term of
        2^-25 times the codes (448 at most) of every key, in the units of the largest weight."""
        G = self.Hq // self.Hkv
        out = torch.zeros((self.N, self.Hq, self.dh), dtype=torch.float64)
        tol = torch.zeros_like(out)
        q, positions, table = self.q.cpu().double(), self.positions.cpu().long(), self.table.cpu().long()
        masks = None if self.masks is None else self.masks.cpu().long()
        sink = None if sink is None else sink.cpu().double()
        slopes = None if slopes is None else slopes.cpu().double()
        at = 0
        for r, (m, c) in enumerate(zip(self.n, self.held)):
            L = m + c
            place = torch.arange(L)
            kv = self.rows[table[r][place // self.page], :, :, place % self.page]  # [L, 2, Hkv, dh]
            for i in range(m):
                p = int(positions[at + i])
                lo = max(p - p % chunk if chunk else 0, p - window + 1 if window else 0)
                key_pos = place.clone()
                if masks is not None:
                    key_pos[c:] = positions[at:at + m]
                    bit = torch.tensor([bool(masks[at + i, j // 32] >> (j % 32) & 1) for j in range(m)], dtype=torch.bool)
                    seen = torch.cat([torch.ones(c, dtype=torch.bool), bit])
                else:
                    seen = place <= p
                seen = seen & (key_pos >= lo)
                if not seen.any():
                    continue
                k, v = kv[seen, 0], kv[seen, 1]
                temp = 1 + temper * math.log1p(math.floor((p + 1) / floor)) if temper else 1.0
                for h in range(self.Hq):
                    x = q[at + i, h]
                    s = k[:, h // G] @ x * self.scale * temp
                    size = float((k[:, h // G].abs() @ x.abs()).max()) * self.scale * temp
                    if cap:
                        s = cap * torch.tanh(s / cap)
                    if slopes is not None:
                        s = s - slopes[h] * (p - key_pos[seen]).double()
                        size += float(slopes[h]) * (p + 1)
                    top = s.max() if sink is None else torch.maximum(s.max(), sink[h])
                    w = torch.exp(s - top)
                    total = w.sum() + (0 if sink is None else torch.exp(sink[h] - top))
                    w = w / total
                    out[at + i, h] = w @ v[:, h // G]
                    A = w @ v[:, h // G].abs()
                    rel = self.weights + 2 * (2 * self.dh * 2.0 ** -24 * size + 2.0 ** -18)
                    tol[at + i, h] = 2.0 ** -8 * out[at + i, h].abs() + rel * A
                    if self.bits8:
                        e = v[:, h // G].abs().amax(-1) / 224  # at least the row's power of two
                        tol[at + i, h] += 2.0 ** -25 * 448 * len(s) * float((w * e).max())
            at += m
        return out, tol


def assert_close(got, want, tol, served=None):
    got = got.detach().cpu().double()
    if served is not None:
        got, want, tol = got[served], want[served], tol[served]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{int(torch.isnan(got).sum())} NaN, {int(torch.isnan(want).sum())} expected"
    off = torch.nan_to_num((got - want).abs() - tol, nan=0.0)
    worst = int(off.argmax())
    assert off.max() <= 0, f"off by {float((got - want).abs().flatten()[worst]):.3e}, allowed {float(tol.flatten()[worst]):.3e} at {worst}"
