"""What rf_lora_workspace_bytes and rf_lora_add_launch make of the numbers of their blocks (no GPU needed)."""
import pytest

from rocmforge_amd import lora

from .test_paged8_args import step, target


def sized(rows=100, num_seqs=2, widths=(512,), in_dim=4096, max_rank=16, num_adapters=3, **kw):
    """Bytes of the workspace of a step of these numbers."""
    s = step(rows=rows, num_seqs=num_seqs, num_adapters=num_adapters, max_rank=max_rank, in_dim=in_dim, ld_x=in_dim, **kw)
    return lora.workspace_bytes(s, [target(a_stride=max_rank * in_dim, b_stride=max_rank * w, ld_base=w, ld_y=w, out_dim=w)
                                    for w in widths])


@pytest.mark.parametrize("rows,num_seqs", [(20, 2), (100, 2), (100, 64), (3000, 200)])
@pytest.mark.parametrize("num_adapters", [63, 64, 65, 1 << 20, (1 << 31) - 1])
def test_as_many_adapters_as_an_integer_counts(rf, rows, num_seqs, num_adapters):
    # requests have 64 adapters at most in a group, so more of them change nothing
    assert sized(rows, num_seqs, num_adapters=num_adapters) == sized(rows, num_seqs, num_adapters=1000) > 0


# what a step can have of each number, rising
SIZES = dict(rows=[1, 4, 5, 16, 63, 64, 100, 767, 768, 1023, 1024, 2559, 2560, 3000, 4607, 4608, 10000, 1 << 17, 1 << 23],
             num_seqs=[1, 2, 64, 65, 200, 5000], widths=[(512,), (512, 1024), (512, 1024, 64)],
             in_dim=[8, 256, 264, 512, 1032, 4096, 12288], max_rank=[8, 16, 24, 32, 40, 64, 72, 128],
             num_adapters=[0, 1, 12, 63, 64, 1000])


@pytest.mark.parametrize("name", SIZES)
def test_no_less_for_more(rf, name):
    # a workspace of a server's largest step serves its smaller ones
    for base in (dict(), dict(rows=3000), dict(num_seqs=200, rows=1000), dict(in_dim=256), dict(max_rank=128, rows=700),
                 dict(widths=(512, 512, 512), rows=2600, in_dim=12288, max_rank=64)):
        got = [sized(**{**base, name: v}) for v in SIZES[name]]
        assert got == sorted(got), (base, got)


@pytest.mark.parametrize("in_dim,max_rank,widths", [(4096, 64, (12288, 12288)), (4096, 16, (4096, 1024, 1024)),
                                                    (12288, 32, (4096,)), (520, 128, (72,)), (264, 8, (64,))])
def test_the_largest_step_s_workspace_serves_all_below(rf, in_dim, max_rank, widths):
    most = sized(5000, 300, widths, in_dim, max_rank, num_adapters=40)
    for rows in list(range(1, 200)) + list(range(200, 5001, 37)) + [767, 768, 2559, 2560]:
        for seqs in (1, 2, 30, 64, 65, 300):
            assert sized(rows, seqs, widths, in_dim, max_rank, num_adapters=40) <= most


def test_it_stays_small(rf):
    # some MB where k is cut, a slot a row and target where there are many
    assert sized(4000, 1, (4096,), 12288, 32) <= 3 << 20
    assert sized(1 << 20, 64, (512, 512, 512), 4096, 64) == 3 * (1 << 20) * 64 * 4
