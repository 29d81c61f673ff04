"""Plain 64-bit attention over a paged cache, and batches to try it on."""
from __future__ import annotations

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Paged:
    """A cache of NaN with the keys and values of some sequences at scattered pages:
    `new` tokens of `total` per sequence."""

    def __init__(self, nxq, new, total, Hq, Hk, D, page, dtype, order="heads", seed=0, fill=math.nan, spare=2, peak=1.0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.new, self.total, self.Hq, self.Hk, self.D, self.page, self.order = new, total, Hq, Hk, D, page, order
        need = [-(-t // page) for t in total]
        pages = sum(need) + spare
        self.shuffled = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
        shape = (pages, Hk, page, D) if order == "heads" else (pages, page, Hk, D)
        self.keys = torch.full(shape, fill, dtype=dtype, device=device)
        self.values = torch.full(shape, fill, dtype=dtype, device=device)
        self.table = torch.full((len(new), max(max(need), 1) + 1), -7, dtype=torch.int32, device=device)
        self.k, self.v, at = [], [], 0  # dense, [total][Hk][D]
        for i, (t, c) in enumerate(zip(total, need)):
            self.table[i, :c] = torch.tensor(self.shuffled[at:at + c], dtype=torch.int32)
            at += c
            k = (peak * torch.randn((t, Hk, D), generator=g, device=device)).to(dtype)
            v = torch.randn((t, Hk, D), generator=g, device=device).to(dtype)
            self.k.append(k)
            self.v.append(v)
        self.store()
        self.T = sum(new)
        self.q = torch.randn((self.T, Hq, D), generator=g, device=device).to(dtype)
        self.q_offsets = torch.tensor([0] + new, device=device).cumsum(0).to(torch.int32)
        self.kv_lens = torch.tensor(total, dtype=torch.int32, device=device)
        self.cache = nxq.KVCache(self.keys, self.values, order=order) if nxq is not None else None

    def places(self, i, n=None):
        j = torch.arange(self.total[i] if n is None else n, device=self.keys.device)
        return self.table[i].long()[j // self.page], j % self.page

    def view(self, x):
        """[pages][slots][heads][D] of the keys or values."""
        return x.transpose(1, 2) if self.order == "heads" else x

    def store(self):
        """Writes the dense keys and values into the pages."""
        for i in range(len(self.total)):
            p, s = self.places(i)
            self.view(self.keys)[p, s] = self.k[i]
            self.view(self.values)[p, s] = self.v[i]

    def attend(self, nxq, **kw):
        return nxq.paged_attention(self.q, self.cache, self.q_offsets, self.kv_lens, self.table, **kw)

    def expected(self, scale=None, window=0, sinks=0, y=None):
        """(out, bound, lse) of every new token in 64 bits, and a bound on |error| but for the output's rounding."""
        scale = self.D ** -0.5 if scale is None else scale
        G, dev = self.Hq // self.Hk, self.q.device
        out = torch.zeros((self.T, self.Hq, self.D), dtype=torch.float64, device=dev)
        bound = torch.zeros_like(out)
        lse = torch.full((self.T, self.Hq), -math.inf, dtype=torch.float64, device=dev)
        u = HALF_STEP[self.q.dtype]
        if y is torch.float32:  # weights as two numbers of the cache's type
            u = u * u
        at = 0
        for i, (n, t) in enumerate(zip(self.new, self.total)):
            k = self.k[i].double().repeat_interleave(G, dim=1).transpose(0, 1)  # [Hq][t][D]
            v = self.v[i].double().repeat_interleave(G, dim=1).transpose(0, 1)
            j = torch.arange(t, device=dev)
            for r0 in range(0, n, 256):
                r1 = min(n, r0 + 256)
                pos = (t - n + torch.arange(r0, r1, device=dev))[:, None]
                see = j <= pos
                if window:
                    see &= (j > pos - window) | (j < sinks)
                q = self.q[at + r0:at + r1].double().transpose(0, 1)
                s = scale * (q @ k.transpose(1, 2))
                mag = scale * (q.abs() @ k.abs().transpose(1, 2))
                s = torch.where(see, s, torch.full_like(s, -math.inf))
                top = s.max(dim=2, keepdim=True)[0] if t else s.new_zeros((self.Hq, r1 - r0, 1))
                top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
                e = torch.where(see, torch.exp(s - top), torch.zeros_like(s))
                z = e.sum(dim=2, keepdim=True)
                zz = torch.where(z == 0, torch.ones_like(z), z)
                clean = torch.where(see.any(dim=0)[None, :, None], v, torch.zeros_like(v))
                o = (e / zz) @ clean
                # Scores: D roundings of a sum, the scale's and the exponent's argument (relative to the
                # magnitude of the terms).  Weights: u each; the exponential 2^-21; sums over t keys.
                ds = torch.where(see, mag, torch.zeros_like(mag)) * (self.D + 8) * 2.0 ** -24
                w = e / zz
                b = (w * (u + 2.0 ** -20 + 2 * ds)) @ clean.abs()
                b += ((w * ds).sum(dim=2, keepdim=True) + (t + 64) * 2.0 ** -23) * (w @ clean.abs())
                if t:  # weights below f16's normal range, 2^-25 of the unit of 2^7
                    b += t * 2.0 ** -32 * clean.abs().amax(dim=1, keepdim=True)
                out[at + r0:at + r1] = o.transpose(0, 1)
                bound[at + r0:at + r1] = b.transpose(0, 1)
                lse[at + r0:at + r1] = torch.where(z > 0, top + torch.log(zz), torch.full_like(z, -math.inf))[..., 0].T
            at += n
        return out, bound, lse

    def check(self, got, lse=None, **kw):
        want, bound, want_lse = self.expected(y=got.dtype, **kw)
        half = HALF_STEP[got.dtype]
        err = (got.double() - want).abs()
        tol = bound * (1 + half) + half * want.abs() + 2.0 ** -24
        ok = (err <= tol) | (torch.isnan(want) & torch.isnan(got.double()))
        assert bool(ok.all()), f"max err/tol {(err / tol).max().item():.3g}, {int((~ok).sum())} of {ok.numel()}"
        if lse is not None:
            fin = torch.isfinite(want_lse)
            assert torch.equal(fin, torch.isfinite(lse))
            # (D + 8) 2^-24 of the terms' magnitude, as above; the magnitude is at most a few times D^0.5.
            assert bool(((lse.double() - want_lse).abs()[fin] <= 2.0 ** -13 + 2.0 ** -20 * want_lse.abs()[fin]).all())
