"""Packed attention where its look-up of sequences takes another way (more than 62 of them), and every head for itself.  Tolerances: test_packed_attention.py."""
import pytest
import torch

from test_packed_attention import check, compare, make, reference, run


def lengths(seed, count, top):
    return torch.randint(0, top, (count,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("table", [None, (16, 20, True)])
@pytest.mark.parametrize("count", [61, 62, 63, 64, 130, 300])
def test_around_the_number_of_lanes(dev, causal, table, count):
    lens = lengths(count, count - 2, 30) + [200, 131]
    compare(make(lens, lens, 4, 2, 64, torch.bfloat16, seed=count, tail=9, lead=2, table=table), dev, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("table", [None, (16, 20, True)])
@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 128), (torch.float16, 40)])
def test_many_with_keys_of_their_own(dev, causal, table, dtype, width):
    """queries and keys of different lengths, some of them none"""
    lq, lk = lengths(1, 100, 20) + [0, 150, 1], lengths(2, 100, 40) + [260, 0, 300]
    d = make(lq, lk, 2, 1, width, dtype, seed=3, tail=5, lead=1, table=table)
    got = compare(d, dev, causal)
    for n in ("o", "dq"):
        assert (got[n][:1] == 0).all() and (got[n][-5:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_many_have_the_bits_of_few(dev, causal):
    """the same sequences in one call of 90 and in calls of 30: outputs and dq have the same bits"""
    lens = [n + 1 for n in lengths(4, 90, 25)]
    d = make(lens, lens, 2, 2, 64, torch.bfloat16, seed=5)
    whole = run(d, dev, causal, cross=False)
    for first in (0, 30, 60):
        rows = slice(sum(lens[:first]), sum(lens[:first + 30]))
        part = {n: d[n][rows] for n in ("q", "k", "v", "do")}
        part["eq"] = torch.tensor([0] + lens[first:first + 30], dtype=torch.int32).cumsum(0, dtype=torch.int32)
        few = run(part, dev, causal, cross=False)
        for n in ("o", "dq"):
            assert torch.equal(few[n], whole[n][rows]), (n, first)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
def test_one_head_at_a_time(dev, causal):
    """a head alone has the bits that it has among others in o, dq and the table's gradient; dk and dv may be shared out among more workgroups and are
    compared with float64"""
    lens = [300, 41, 129]
    d = make(lens, lens, 4, 4, 64, torch.bfloat16, seed=12, table=(32, 64, True))
    joint = run(d, dev, causal, cross=False)
    for h in range(4):
        one = {n: (t[:, h:h + 1] if t.dim() == 3 else t) for n, t in d.items()}
        one["table"] = d["table"][:, h:h + 1].contiguous()
        got = run(one, dev, causal, cross=False)
        for n in ("o", "dq", "dtable"):
            assert torch.equal(got[n], joint[n][:, h:h + 1]), (n, h)
        want, tol = reference(one, causal)
        for n in ("dk", "dv"):
            check(n, got[n], want[n], tol[n])
