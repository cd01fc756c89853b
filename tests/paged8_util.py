"""8-bit pages for the GPU tests: e4m3 by a table of its values in float64, and the
pages' exponents, from their definition."""
import math

import torch

from rocmforge_amd import paged

from . import paged_util as P

DEV = P.DEV
E_LO, E_HI = -15, 7
NAN = 0x7f


def table():
    """The values of the codes 0 .. 126, rising."""
    return [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]


def values(codes, exponents, block):
    """float64 of codes [pages][page][heads][d] under exponents [pages][page / block][heads] (+ 127)."""
    t = torch.tensor(table() + [math.nan], dtype=torch.float64, device=codes.device)
    c = codes.long()
    x = torch.where(c >= 128, -t[c & 127], t[c & 127])
    e = exponents.long().clamp(E_LO + 127, E_HI + 127) - 127
    return x * torch.exp2(e.double()).repeat_interleave(block, 1)[..., None]


def exponent(amax):
    """The smallest e in [-15, 7] with amax <= 448 2^e, 7 where there is none."""
    out = torch.full(amax.shape, E_HI, dtype=torch.int64, device=amax.device)
    for e in range(E_HI, E_LO - 1, -1):
        out = torch.where(amax.double() <= 448.0 * 2.0 ** e, e, out)
    return out


def nearest(x):
    """Codes of float64 values: the nearest, ties to the even code; beyond 448 448, NaN of what is not finite."""
    t = torch.tensor(table(), dtype=torch.float64, device=x.device)
    mid = (t[1:] + t[:-1]) / 2
    a = x.abs().clamp(max=448.0)
    i = torch.searchsorted(mid, a.nan_to_num(0.0).contiguous())          # mid[i - 1] < a <= mid[i]
    tie = (i < 126) & (mid[i.clamp(max=125)] == a)
    i = i + (tie & (i % 2 == 1))
    i = torch.where(x.isfinite(), i, NAN)
    return torch.where(torch.signbit(x), i | 128, i).to(torch.uint8)


class Pages:
    """Codes and exponents in pages, [page][row][head][d] to look at, by_head: heads outside the rows in memory;
    extra: bytes between one head's row and the next.  Filled with NaN, and exponents of no meaning."""

    def __init__(self, pages, page, nkv, d, by_head=False, extra=0):
        self.block, self.page = min(page, 16), page
        shape = (pages, nkv, page, d + extra) if by_head else (pages, page, nkv, d + extra)
        mk = lambda: torch.full(shape, NAN, dtype=torch.uint8, device=DEV)[..., :d]
        self.k, self.v = [t.transpose(1, 2) if by_head else t for t in (mk(), mk())]
        self.ks, self.vs = [torch.full((pages, page // self.block, nkv), 255, dtype=torch.uint8, device=DEV)
                            for _ in range(2)]

    def cache(self):
        pages, page, nkv, d = self.k.shape
        return paged.PagedCache8(k=self.k, v=self.v, k_scale=self.ks, v_scale=self.vs, page_stride=self.k.stride(0),
                                 row_stride=self.k.stride(1), head_stride=self.k.stride(2), num_pages=pages,
                                 page_size=page, num_kv_heads=nkv, head_dim=d)

    def values(self):
        """(k, v) in float64."""
        return [values(c, e, self.block) for c, e in ((self.k, self.ks), (self.v, self.vs))]

    def hold(self, k, v):
        """Takes fp16 pages in: what is not NaN is rounded, and its blocks get the exponents they need."""
        for x, codes, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
            x = x.double()
            pages, page, nkv, d = x.shape
            top = x.abs().nan_to_num(0.0, 0.0).view(pages, page // self.block, self.block, nkv, d).amax((2, 4))
            e = exponent(top)
            scale.copy_(e + 127)
            codes.copy_(nearest(x * torch.exp2(-e.double()).repeat_interleave(self.block, 1)[..., None]))
