"""The rotary step into the pages (rf_paged_rope_write_launch) and its table of
turns against float64."""
import math

import pytest
import torch

from rocmforge_amd import paged

from . import paged_util as P

pytestmark = pytest.mark.gpu


def turns64(rot, base, mode=paged.ROPE_PLAIN, factor=1.0, orig=0.0, fast=32.0, slow=1.0, scale=None):
    out = []
    for i in range(rot // 2):
        th = base ** (-2.0 * i / rot) / (scale[i] if scale else 1.0)
        if mode == paged.ROPE_LINEAR:
            th /= factor
        if mode == paged.ROPE_YARN:
            pair = lambda beta: rot * math.log(orig / (2 * math.pi * beta)) / (2 * math.log(base))
            lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
            r = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            th = th * (1 - r) + th / factor * r
        out.append(th / (2 * math.pi))
    return torch.tensor(out, dtype=torch.float64, device=P.DEV)


@pytest.mark.parametrize("rot", [2, 16, 20, 64, 128, 256])
@pytest.mark.parametrize("base", [1e4, 5e5, 1e6])
@pytest.mark.parametrize("kw", [dict(), dict(mode=1, factor=8.0), dict(mode=2, factor=4.0, orig=32768.0),
                                dict(mode=2, factor=40.0, orig=4096.0, fast=32.0, slow=1.0),
                                dict(mode=2, factor=2.0, orig=8.0), dict(scale=True)])
def test_turns(rf, dev, rot, base, kw):
    kw = dict(kw)
    scale = None
    if kw.pop("scale", False):
        scale = [float(torch.tensor(1.0 + 0.37 * i).float()) for i in range(rot // 2)]
    t = torch.zeros(rot // 2 + 1, dtype=torch.float64, device=P.DEV)
    fs = torch.tensor(scale, device=P.DEV) if scale else None
    paged.rope_turns_table(t, rot, base, kw.get("mode", 0), kw.get("factor", 1.0), kw.get("orig", 0.0),
                           kw.get("fast", 32.0), kw.get("slow", 1.0), fs)
    torch.cuda.synchronize()
    want = turns64(rot, base, scale=scale, **kw)
    assert bool(((t[:-1] - want).abs() <= 1e-13 * want).all()) and t[-1].item() == 0.0


class Step:
    def __init__(self, slots, pos, nh=4, nkv=2, d=128, rot=None, neox=1, norm=True, page=16, pages=8, by_head=False,
                 extra=0, wide=0, factor=1.0, base=1e6, seed=0):
        g = P.gen(seed + 31 * len(slots) + d)
        rows, rot = len(slots), d if rot is None else rot
        mk = lambda n: torch.randn(rows, n * d + wide, generator=g, device=P.DEV)[:, :n * d]
        self.q, self.k, self.v = mk(nh), mk(nkv), mk(nkv)
        w = lambda: 1 + 0.2 * torch.randn(d, generator=g, device=P.DEV) if norm else None
        self.qn, self.kn = w(), w()
        self.kc, self.vc = P.cache_tensors(pages, page, nkv, d, by_head, extra)
        self.kc.fill_(9.0)
        self.vc.fill_(9.0)
        self.q16 = torch.full((rows, nh * d + 8), 9.0, dtype=torch.float16, device=P.DEV)
        self.turns = turns64(rot, base) if rot else torch.zeros(1, dtype=torch.float64, device=P.DEV)
        self.pos, self.slot = P.ints(pos), P.ints(slots)
        self.cache = P.cache_block(self.kc, self.vc)
        self.dims = (rows, nh, nkv, d, rot, neox, page, factor)
        self.args = paged.PagedRope(q=self.q, k=self.k, v=self.v, q_norm=self.qn, k_norm=self.kn, q16=self.q16,
                                    positions=self.pos, slots=self.slot, turns=self.turns, ld_q=self.q.stride(0),
                                    ld_k=self.k.stride(0), ld_v=self.v.stride(0), ld_q16=self.q16.stride(0), rows=rows,
                                    num_heads=nh, rot_dim=rot, neox=neox, eps=1e-6, attn_factor=factor)

    def turned(self, x, w):
        """(value, size of its pair) of every element, float64."""
        rows, nh, nkv, d, rot, neox, page, factor = self.dims
        x = x.double().reshape(rows, -1, d)
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        if rot == 0:
            return x, x.abs()
        ang = 2 * math.pi * (self.pos.double()[:, None] * self.turns)[:, None, :]
        c, s = ang.cos() * factor, ang.sin() * factor
        i = torch.arange(rot // 2, device=P.DEV)
        i0, i1 = (i, i + rot // 2) if neox else (2 * i, 2 * i + 1)
        y, size = x.clone(), x.abs()
        y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i0] * s + x[..., i1] * c
        size[..., i0] = size[..., i1] = (x[..., i0].abs() + x[..., i1].abs()) * factor
        return y, size

    def run(self):
        print(f"[gpu] rope write {self.dims}", flush=True)
        paged.rope_write(self.args, self.cache)
        torch.cuda.synchronize()

    def check(self):
        rows, nh, nkv, d, rot, neox, page, factor = self.dims
        total = self.kc.shape[0] * page
        self.run()
        live = (self.slot >= 0) & (self.slot < total)
        at = self.slot[live].long()

        def near(got, want, size):
            # one fp16 rounding, and a few fp32 ones of the pair's size: norm 4, angle (2^-22 of a
            # radian and its cosine and sine) 4, rotation 3, each at most 2^-23
            bound = P.U16 * want.abs() + 2.0 ** -25 + 11 * 2.0 ** -23 * size
            assert bool(((got.double() - want).abs() <= bound).all()), \
                ((got.double() - want).abs() / bound).max().item()

        want, size = self.turned(self.q, self.qn)
        near(self.q16[live][:, :nh * d].reshape(-1, nh, d), want[live], size[live])
        assert bool((self.q16[~live] == 9.0).all()) and bool((self.q16[:, nh * d:] == 9.0).all())
        want, size = self.turned(self.k, self.kn)
        near(self.kc[at // page, at % page], want[live], size[live])
        v = self.v.reshape(rows, nkv, d)[live].half()
        assert torch.equal(self.vc[at // page, at % page], v)
        rest = torch.ones(self.kc.shape[:2], dtype=torch.bool, device=P.DEV)
        rest[at // page, at % page] = False
        assert bool((self.kc[rest] == 9.0).all()) and bool((self.vc[rest] == 9.0).all())


@pytest.mark.parametrize("d,rot", [(64, 64), (64, 16), (128, 128), (128, 64), (128, 96), (128, 8), (128, 0), (256, 256),
                                   (256, 64)])
@pytest.mark.parametrize("neox", [0, 1])
@pytest.mark.parametrize("norm", [False, True])
def test_layouts(rf, dev, d, rot, neox, norm):
    Step([5, 100, 17, 0, 127], [0, 1, 77, 4000, 131071], d=d, rot=rot, neox=neox, norm=norm).check()


@pytest.mark.parametrize("nh,nkv", [(1, 1), (3, 3), (32, 8), (28, 4), (40, 1), (64, 8)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_head_counts(rf, dev, nh, nkv, d):
    Step([3], [9], nh, nkv, d).check()
    Step(list(range(70, 0, -1)), list(range(500, 570)), nh, nkv, d, page=8, pages=9).check()


@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("page", [8, 64, 1024])
def test_pages_strides_and_padding(rf, dev, page, by_head):
    slots = [page * 2 + 1, -1, 0, page * 3 - 1, -1, page - 1, page * 3, 2 ** 31 - 1, -2 ** 31]
    Step(slots, list(range(9)), page=page, pages=3, by_head=by_head, extra=16, wide=12).check()


def test_many_rows(rf, dev):
    Step(list(range(2999, -1, -1)), list(range(60000, 63000)), nh=8, nkv=2, page=16, pages=188).check()


@pytest.mark.parametrize("pos", [0, 1, 1000, 131072, 10 ** 7, 2 ** 31 - 1, -5])
@pytest.mark.parametrize("base", [1e4, 1e6])
def test_far_positions(rf, dev, pos, base):
    Step([1, 2], [pos, pos], base=base, norm=False).check()


def test_scaled_rotation_and_large_values(rf, dev):
    Step([1, 2, 3], [7, 70, 700], factor=1.1386).check()
    s = Step([1, 2, 3], [7, 70, 700], norm=False)
    s.q *= 1e6                     # beyond fp16: infinities, as a conversion gives
    s.run()
    want, _ = s.turned(s.q, None)
    far = want.abs() > 70000
    assert bool(s.q16[:, :512].reshape(3, 4, 128)[far].isinf().all())


def test_one_norm_only(rf, dev):
    s = Step([1, 2], [3, 4])
    s.kn = None
    s.args.k_norm = None
    s.check()


def test_the_same_step_as_the_row_launcher(rf, dev):
    """rf_qk_norm_rope_kv_write_rows on a contiguous cache: the same values but for
    the angle's fp32 rounding."""
    import ctypes

    from . import gpu_util as G
    rows, nh, nkv, d = 50, 8, 2, 128
    s = Step(list(range(16, 66)), list(range(rows)), nh, nkv, d, pages=5)
    s.check()
    q16 = torch.zeros(rows, nh * d, dtype=torch.float16, device=P.DEV)
    kc, vc = [torch.zeros(64, nkv, d, dtype=torch.float16, device=P.DEV) for _ in range(2)]
    G.call(rf.rf_qk_norm_rope_kv_write_rows, G.ptr(s.q), G.ptr(s.k), G.ptr(s.v), G.ptr(s.qn), G.ptr(s.kn), G.ptr(q16),
           G.ptr(kc), G.ptr(vc), 0, rows, rows, nh, nkv, d, 64, 1e-6, ctypes.c_float(1e6), 1, None, None, None)
    # angles below 50: off by 2^-19 there, and a rounding to fp16 on each side
    got = s.kc.reshape(-1, nkv, d)[16:66].double()
    assert bool(((got - kc[:rows].double()).abs() <= 2 * P.U16 * got.abs() + 2.0 ** -17 * 6).all())
    assert torch.equal(s.vc.reshape(-1, nkv, d)[16:66], vc[:rows])
    got = s.q16[:, :nh * d].double()
    assert bool(((got - q16.double()).abs() <= 2 * P.U16 * got.abs() + 2.0 ** -17 * 6).all())
