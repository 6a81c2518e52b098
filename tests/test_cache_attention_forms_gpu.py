"""The forms of the paged attention kernel (one band or two, sets of two or four heads, wide values) against 64 bits; tolerances are
those of tests/test_cache_pages_gpu.py, derived there for one rounding of the folded query: the two-band form's further roundings
(the coefficients and the folded rows, of the low pairs alone) have to stay within its six standard deviations as well."""
import pytest
import torch

from . import test_cache_pages_gpu as pages

pytestmark = pytest.mark.gpu

SHAPES = [dict(lens=[260, 31, 0, 1], Rk=8, Rv=8), dict(lens=[300, 129], Rk=24, Rv=136), dict(lens=[500], Rk=64, Rv=192, gs=3),
          dict(lens=[260, 31], Rk=96, Rv=392, P=32), dict(lens=[700, 5], Rk=128, Rv=512, P=64), dict(lens=[300], Rk=72, Rv=456, gs=8, G=1),
          dict(lens=[385, 128, 2], Rk=256, Rv=448), dict(lens=[1000], Rk=104, Rv=384, gs=5)]


def _at(case, theta, monkeypatch):
    from palu_amd.kernel import paged
    monkeypatch.setattr(pages, "THETA", theta)
    return paged.paged_attn(*case.args(), theta=theta)


@pytest.mark.parametrize("theta", [100.0, 8300.0, 8500.0, 5e5])
@pytest.mark.parametrize("kw", SHAPES, ids=str)
def test_frequencies_on_both_sides_of_the_two_band_rule(kw, theta, monkeypatch):
    """64 f_32 is 6.4, 0.7025, 0.694 and 0.09 rad: one band up to 8400"""
    case = pages.Case(**kw)
    case.check(_at(case, theta, monkeypatch))


@pytest.mark.parametrize("kw", SHAPES, ids=str)
def test_a_table_that_is_not_registered_takes_one_band(kw, monkeypatch):
    from palu_amd.kernel import paged
    table = paged.rope_inv_freq
    monkeypatch.setattr(paged, "rope_inv_freq", lambda *a: table(*a).clone())
    case = pages.Case(**kw)
    case.check(paged.paged_attn(*case.args()))


@pytest.mark.parametrize("Rk,Rv,gs", [(64, 192, 4), (128, 384, 4), (128, 512, 4), (64, 64, 2)])
@pytest.mark.parametrize("where", [0, 5, 1 << 20, (1 << 30) - 1, -4000])
def test_queries_far_from_their_rows(Rk, Rv, gs, where):
    """the query's position has nothing to do with the rows': angles of a million positions, in front of them and behind"""
    case = pages.Case([400, 130], Rk=Rk, Rv=Rv, gs=gs)
    case.qpos = torch.tensor([where, where // 2], dtype=torch.int32)
    case.check(pages._run(case))


@pytest.mark.parametrize("Rk,Rv", [(64, 192), (128, 384), (128, 512)])
def test_long_sequences_cut_into_many_pieces(Rk, Rv):
    """pieces that begin at odd and even tiles, in the middle of a sequence and across the ends of several"""
    case = pages.Case([9000, 130, 0, 4097, 1, 2500, 128], G=3, Rk=Rk, Rv=Rv, P=64)
    case.check(pages._run(case))
