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


def test_more_sequences_than_the_plan_reads_at_once():
    """a thousand sequences: every workgroup finds its piece in sixteen rounds of 64 lengths"""
    case = pages.Case([(53 * i * i + 7 * i) % 290 if i % 5 else 0 for i in range(1000)], gs=1, G=1, Rk=32, Rv=32)
    case.check(pages._run(case))


def test_calls_with_nothing_in_them():
    from palu_amd.kernel import paged
    pool = paged.make_pool(2, 2, 16, 64, 96)
    frag = paged.prepare_paged_b(torch.zeros(8, 64, 128).half().cuda(), 2)
    i32 = dict(dtype=torch.int32, device="cuda")
    assert paged.paged_attn(torch.zeros(0, 8, 128).half().cuda(), frag, pool, torch.zeros(0, 3, **i32), torch.zeros(0, **i32)).shape == (0, 8, 96)
    q = torch.ones(2, 8, 128).half().cuda()
    out = paged.paged_attn(q, frag, pool, torch.zeros(2, 0, **i32), torch.tensor([0, 3], **i32))
    assert bool((out[0] == 0).all()) and bool(out[1].isnan().all())          # a length that the table has no room for
    before = [t.clone() for t in pool]
    none = torch.zeros(0, **i32)
    paged.paged_append(pool, torch.zeros(0, 2, 64).half().cuda(), torch.zeros(0, 2, 96).half().cuda(), torch.zeros(2, 1, **i32), none, none)
    one = torch.zeros(1, **i32)
    paged.paged_append(pool, torch.ones(1, 2, 64).half().cuda(), torch.ones(1, 2, 96).half().cuda(), torch.zeros(2, 0, **i32), one, one)
    paged.paged_copy(pool, none, none)
    paged.paged_copy(pool, [], [])
    assert all(torch.equal(a, b) for a, b in zip(pool, before))


@pytest.mark.parametrize("Rk,gs", [(64, 4), (64, 2), (192, 4)])
def test_a_query_that_is_not_finite_spoils_its_head_only(Rk, gs):
    case = pages.Case([200, 40], Rk=Rk, gs=gs)
    good = pages._run(case)
    case.q[0, 1, 5], case.q[1, 2, 100] = float("nan"), float("inf")
    out = pages._run(case)
    spoilt = torch.zeros(2, case.H, dtype=torch.bool)
    spoilt[0, 1] = spoilt[1, 2] = True
    assert bool(out[spoilt].isnan().all()) and torch.equal(out[~spoilt], good[~spoilt])


def test_scores_of_another_scale():
    from palu_amd.kernel import paged
    case = pages.Case([300, 17])
    same = paged.paged_attn(*case.args(), sm_scale=128 ** -0.5)
    assert torch.equal(same, pages._run(case))
    case.q *= 4                                                              # (a power of two: the same roundings)
    assert torch.equal(paged.paged_attn(*case.args(), sm_scale=128 ** -0.5 / 4), same)


def test_sequences_that_share_all_their_pages():
    """the same rows under several table rows, one query each: what one sequence gives, for every one"""
    from palu_amd.kernel import paged
    case = pages.Case([700], Rk=128, Rv=384, P=64)
    q, frag, pool, table, lens, pos = case.args()
    qs = torch.cat([q, q * 0.5, q, q * 2])
    many = paged.paged_attn(qs, frag, pool, table.expand(4, -1), lens.expand(4).contiguous(), pos.expand(4).contiguous())
    ref, tol = case.reference()
    for i in (0, 2):
        assert bool(((many[i].double() - ref[0]).abs() <= tol[0]).all())
    assert not torch.equal(many[1], many[0])
