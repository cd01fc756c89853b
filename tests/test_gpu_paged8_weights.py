"""The weights of the attention over 8-bit pages: a row of one key."""
import pytest
import torch

from . import paged_util as P
from .test_gpu_paged8_attn import Case


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("out_f32", [0, 1])
@pytest.mark.parametrize("new,kv", [(1, 1), (1, 300), (3, 40), (5, 5), (40, 700), (200, 200)])
def test_a_row_of_one_key_is_its_value(rf, dev, d, out_f32, new, kv):
    # o / l with o = w v exact: a reciprocal and a product, 2^-24 each; v itself is one of fp16's values
    c = Case([new], [kv], window=1, d=d, out_f32=out_f32, sizes=8.0)
    got = c.run()
    t = torch.arange(kv - new, kv, device=P.DEV)
    v = c.v[c.tab[0].long()[t // 16], t % 16].double().repeat_interleave(c.nh // c.v.shape[2], 1)
    assert bool(((got - v).abs() <= (v.abs() * 2.0 ** -23 if out_f32 else 0.0)).all())
    # the first row of a prompt sees one key without a window too
    c.args.window = 0
    if new == kv:
        assert bool(((c.run()[0] - v[0]).abs() <= (v[0].abs() * 2.0 ** -23 if out_f32 else 0.0)).all())
