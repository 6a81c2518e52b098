"""Pages of the 4-bit latent cache on the GPU: rows written into pages, pages copied, and the attention that reads them, each against
a plain evaluation in 64 bits.

Tolerance of the attention (computed per case, before the kernel's result is looked at): with x the latents, F the query folded into
B and rounded to fp16 (half a step = 2^-11 of each element), the score of a position is a sum of independent products x F T, so its
error has a standard deviation below 2^-11 / sqrt(3) * sqrt(sum (x F T)^2) <= 2^-11 / sqrt(3) * |x|_rms-weighted norm; six of those
are granted, `d`.  A softmax whose scores are off by at most d is off by a factor within exp(+-2 d).  The weights are rounded to fp16
once more (2^-11 each, of either sign) and the result once (2^-11 of its value):
    |ctx - ref| <= (exp(2 d) - 1 + 2^-11) sum p |v| + 2^-11 |ref|  (+ half the smallest fp16 step)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
THETA = 10000.0


def _inv_freq():
    return (1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D))).double()


class Case:
    """A random pool with B sequences in it.  Rows and pages that belong to nobody hold codes of 15 and NaN pairs."""

    def __init__(self, lens, gs=4, G=2, Rk=64, Rv=96, P=16, seed=0, rotated=False, spare=3, table_pad=2, q_std=2.0, zeros_int=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.gs, self.G, self.Rk, self.Rv, self.P, self.rotated = list(lens), gs, G, Rk, Rv, P, rotated
        self.H, self.B = gs * G, len(lens)
        need = [(n + P - 1) // P for n in lens]
        self.N = sum(need) + spare
        order = torch.randperm(self.N, generator=g).tolist()
        M = max(need + [1]) + table_pad
        table = torch.full((self.B, M), -7, dtype=torch.int32)                # entries past the end name no page
        self.kc = torch.full((self.N, G, P, Rk // 2), 255, dtype=torch.uint8)
        self.vc = torch.full((self.N, G, P, Rv // 2), 255, dtype=torch.uint8)
        self.km = torch.full((self.N, G, P, 2), float("nan"), dtype=torch.float16)
        self.vm = torch.full((self.N, G, P, 2), float("nan"), dtype=torch.float16)
        self.k, self.v = [], []                                               # values in 64 bits, [G, n, R]
        at = 0
        for b, n in enumerate(lens):
            pages = order[at:at + need[b]]
            at += need[b]
            table[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
            for codes, meta, R, out in ((self.kc, self.km, Rk, self.k), (self.vc, self.vm, Rv, self.v)):
                c = torch.randint(0, 16, (G, n, R), generator=g)
                s = (torch.rand((G, n), generator=g) * 0.2 + 0.05).half()
                z = torch.randint(0, 16, (G, n), generator=g).half() if zeros_int else (torch.rand((G, n), generator=g) * 15).half()
                out.append((c.double() - z.double()[..., None]) * s.double()[..., None])
                packed = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
                for j, page in enumerate(pages):
                    m = min(P, n - j * P)
                    codes[page, :, :m] = packed[:, j * P:j * P + m]
                    meta[page, :, :m, 0] = s[:, j * P:j * P + m]
                    meta[page, :, :m, 1] = z[:, j * P:j * P + m]
        self.table = table
        self.q = (torch.randn((self.B, self.H, D), generator=g) * q_std).half()
        self.b = (torch.randn((self.H, Rk, D), generator=g) * Rk ** -0.5 * 0.5).half()
        self.qpos = torch.tensor([max(n - 1, 0) for n in lens], dtype=torch.int32)

    def pool(self):
        from palu_amd.kernel import paged
        return paged.PagePool(self.kc.cuda(), self.km.cuda(), self.vc.cuda(), self.vm.cuda())

    def args(self):
        from palu_amd.kernel import paged
        lens = torch.tensor(self.lens, dtype=torch.int32).cuda()
        return (self.q.cuda(), paged.prepare_paged_b(self.b.cuda(), self.G), self.pool(), self.table.cuda(), lens,
                None if self.rotated else self.qpos.cuda())

    def reference(self):
        """-> (ctx, allowed error), both [B, H, Rv] in 64 bits on the GPU"""
        inv = _inv_freq().cuda()
        ref = torch.zeros((self.B, self.H, self.Rv), dtype=torch.float64, device="cuda")
        tol = torch.full_like(ref, 2.0 ** -25)
        for b, n in enumerate(self.lens):
            if n == 0:
                continue
            x, v = self.k[b].cuda(), self.v[b].cuda()
            q = self.q[b].double().cuda()
            if not self.rotated:
                a = float(self.qpos[b]) * inv
                q = torch.cat((q[:, :64] * a.cos() - q[:, 64:] * a.sin(), q[:, 64:] * a.cos() + q[:, :64] * a.sin()), -1)
            a = torch.arange(n, device="cuda").double()[:, None] * inv
            c, s = a.cos(), a.sin()
            for h in range(self.H):
                g = h // self.gs
                bm = self.b[h].double().cuda()
                key = x[g] @ bm
                rot = torch.cat((key[:, :64] * c - key[:, 64:] * s, key[:, 64:] * c + key[:, :64] * s), -1)
                sc = (rot @ q[h]) / math.sqrt(D)
                p = torch.softmax(sc, -1)
                ref[b, h] = p @ v[g]
                # sum over r, i of (x_r F_ri T_i)^2 <= x^2 . sum_i (|q_i| |b_ri| + |q_i'| |b_ri'|)^2
                qa, ba = q[h].abs(), bm.abs()
                f = (qa[:64] * ba[:, :64] + qa[64:] * ba[:, 64:]) ** 2 + (qa[64:] * ba[:, :64] + qa[:64] * ba[:, 64:]) ** 2
                d = 6 * 2.0 ** -11 / math.sqrt(3) * float(((x[g] ** 2) @ f.sum(-1)).max().sqrt()) / math.sqrt(D)
                tol[b, h] += (math.exp(2 * d) - 1 + 2.0 ** -11) * (p @ v[g].abs()) + 2.0 ** -11 * ref[b, h].abs()
        return ref, tol

    def check(self, ctx):
        ref, tol = self.reference()
        assert ctx.shape == ref.shape and ctx.dtype == torch.float16
        worst = ((ctx.double() - ref).abs() / tol).max().item()
        assert worst <= 1.0, worst


def _run(case):
    from palu_amd.kernel import paged
    return paged.paged_attn(*case.args())


# ------------------------------------------------------------------------------------------------------------ rows into pages
def _exact_quantise(x):
    """quantize_tensor's defaults in 64 bits with its fp16 roundings -> (codes, scale, zero)"""
    def h(t):
        return t.astype(np.float16).astype(np.float64)
    w = x.numpy().astype(np.float64)
    low, high = w.min(-1, keepdims=True), w.max(-1, keepdims=True)
    scale = h(np.maximum(h(high - low), float(np.float16(1e-5))) / 15)
    zero = np.clip(np.rint(h(-low / scale)), 0, 15)
    return np.clip(h(np.rint(h(w / scale)) + zero), 0, 15).astype(np.uint8), scale[..., 0], zero[..., 0]


@pytest.mark.parametrize("Rk,Rv,G,P,lens,skip", [
    (32, 32, 1, 16, [1], 0), (8, 8, 3, 16, [5, 40], 3), (40, 72, 5, 16, [17, 1, 16, 31], 7), (128, 384, 8, 64, [130, 63], 0),
    (256, 512, 2, 128, [129], 1), (64, 192, 8, 32, [1] * 33, 0), (104, 136, 2, 64, [200], 5)])
def test_append_writes_exactly_the_quantised_rows(Rk, Rv, G, P, lens, skip):
    from palu_amd.kernel import paged, quant
    g = torch.Generator().manual_seed(Rk + Rv)
    starts = [int(v) for v in torch.randint(0, 2 * P, (len(lens),), generator=g)]
    need = [(a + n + P - 1) // P for a, n in zip(starts, lens)]
    N = sum(need) + 2
    order = torch.randperm(N, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)] + [torch.full((skip,), -1)]).to(torch.int32)
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(starts, lens)] + [torch.arange(skip)]).to(torch.int32)
    mix = torch.randperm(seq.numel(), generator=g)
    seq, pos = seq[mix], pos[mix]
    T = seq.numel()
    pool = paged.make_pool(N, G, P, Rk, Rv)
    for t in pool:
        t.fill_(9)
    before = [t.cpu() for t in pool]
    # rows of a wider tensor (strides), of very different sizes, some constant, some of one sign
    k = torch.randn((T, G, Rk), generator=g) * torch.exp(3 * torch.randn((T, G, 1), generator=g))
    v = torch.randn((T, G, Rv), generator=g) * torch.exp(3 * torch.randn((T, G, 1), generator=g))
    k[::5] = 0.25
    v[1::7] = v[1::7].abs() + 1
    v[2::7] = -v[2::7].abs() - 1
    k, v = k.clamp(-6e4, 6e4).half(), v.clamp(-3e4, 3e4).half()
    wide = torch.zeros((T, G, Rk + Rv + 8), dtype=torch.float16, device="cuda")
    wide[..., :Rk], wide[..., Rk:Rk + Rv] = k.cuda(), v.cuda()
    paged.paged_append(pool, wide[..., :Rk], wide[..., Rk:Rk + Rv], table.cuda(), seq.cuda(), pos.cuda())
    ok = (seq >= 0).numpy()
    page, off = table[seq[ok].long(), pos[ok].long() // P].long(), pos[ok].long() % P
    for (codes, meta), (c0, m0), x in (((pool.k_codes, pool.k_meta), before[:2], k), ((pool.v_codes, pool.v_meta), before[2:], v)):
        c, s, z = _exact_quantise(x[ok])
        want_c, want_m = c0.clone(), m0.clone()
        want_c[page, :, off] = torch.from_numpy(c[..., 0::2] | (c[..., 1::2] << 4))
        want_m[page, :, off, 0] = torch.from_numpy(s).half()
        want_m[page, :, off, 1] = torch.from_numpy(z).half()
        assert torch.equal(codes.cpu(), want_c) and torch.equal(meta.cpu(), want_m)
    if Rk % 8 == 0:
        cc, mm = quant.quantize_pack(k.cuda(), 4)
        assert torch.equal(pool.k_codes[page.cuda(), :, off.cuda()], cc[ok]) and torch.equal(pool.k_meta[page.cuda(), :, off.cuda()], mm[ok])


def test_append_of_extreme_rows_equals_the_framework_quantiser():
    """subnormals, the ends of fp16, infinities and NaN: the same bits as `quantize_pack`"""
    from palu_amd.kernel import paged, quant
    G, R, P = 2, 64, 16
    g = torch.Generator().manual_seed(3)
    rows = [torch.zeros(R), torch.full((R,), 65504.0), torch.full((R,), -65504.0), torch.randn(R, generator=g) * 1e-7,
            torch.randn(R, generator=g) * 6e4, torch.randn(R, generator=g).sign() * 65504, torch.randn(R, generator=g) * 2e-5,
            torch.arange(R).float(), -torch.arange(R).float(), torch.randn(R, generator=g)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.randn(R, generator=g)
        r[5] = bad
        rows.append(r)
    x = torch.stack(rows).clamp(-65504, 65504).half()
    x[-3, 5], x[-2, 5], x[-1, 5] = float("inf"), float("-inf"), float("nan")
    x = x[:, None].repeat(1, G, 1).cuda()
    T = x.shape[0]
    pool = paged.make_pool(1, G, P, R, R)
    i = torch.arange(T, dtype=torch.int32, device="cuda")
    paged.paged_append(pool, x, x, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros_like(i), i)
    c, m = quant.quantize_pack(x, 4)
    assert torch.equal(pool.k_codes[0, :, :T], c.transpose(0, 1)) and torch.equal(pool.v_codes[0, :, :T], c.transpose(0, 1))
    a, b = pool.k_meta[0, :, :T].view(torch.int16), m.transpose(0, 1).contiguous().view(torch.int16)
    same = (a == b) | (pool.k_meta[0, :, :T].isnan() & m.transpose(0, 1).isnan())
    assert same.all()


def test_append_skips_rows_that_have_no_place():
    from palu_amd.kernel import paged
    G, R, P, N = 1, 32, 16, 3
    pool = paged.make_pool(N, G, P, R, R)
    before = [t.clone() for t in pool]
    table = torch.tensor([[0, 99], [-1, 2]], dtype=torch.int32, device="cuda")
    #       unknown sequence, negative position, past the table, page outside the pool, no page
    seq = torch.tensor([2, 0, 0, 0, 1, -1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, -1, 32, 16, 0, 0], dtype=torch.int32, device="cuda")
    x = torch.randn((6, G, R), device="cuda").half()
    paged.paged_append(pool, x, x, table, seq, pos)
    assert all(torch.equal(a, b) for a, b in zip(pool, before))
    paged.paged_append(pool, x[:0], x[:0], table, seq[:0], pos[:0])
    paged.paged_append(pool, x, x, table[:, :0], seq, pos)


# ------------------------------------------------------------------------------------------------------------------- copies
def _random_pool(N, G, P, Rk, Rv, layers, seed):
    from palu_amd.kernel import paged
    pool = paged.make_pool(N, G, P, Rk, Rv, layers)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in pool:
        if t.dtype == torch.uint8:
            t.random_(0, 256, generator=g)
        else:
            t.normal_(generator=g)
    return pool


@pytest.mark.parametrize("N,G,P,Rk,Rv,layers,n", [(4, 1, 16, 8, 8, None, 1), (9, 5, 16, 40, 72, 3, 4), (40, 8, 64, 128, 384, 2, 20),
                                                  (7, 3, 128, 256, 512, None, 3), (64, 2, 32, 104, 24, 5, 32)])
def test_copy_moves_whole_pages_and_nothing_else(N, G, P, Rk, Rv, layers, n):
    from palu_amd.kernel import paged
    order = torch.randperm(N, generator=torch.Generator().manual_seed(n)).tolist()
    src, dst = order[:n], order[n:2 * n]
    src[-1] = src[0]                                                          # one page copied twice
    for as_tensor in (False, True):
        pool = _random_pool(N, G, P, Rk, Rv, layers, 1)
        want = [t.clone() for t in pool]
        for t in want:
            for a, b in zip(src, dst):
                t[..., b, :, :, :] = t[..., a, :, :, :]
        if as_tensor:
            paged.paged_copy(pool, torch.tensor(src, dtype=torch.int32).cuda(), torch.tensor(dst, dtype=torch.int32).cuda())
        else:
            paged.paged_copy(pool, src, dst)
        for a, b in zip(pool, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_copy_refuses_or_skips_what_it_cannot_do():
    from palu_amd.kernel import paged
    pool = _random_pool(4, 1, 16, 32, 32, None, 2)
    before = [t.clone() for t in pool]
    for src, dst in (([0], [4]), ([-1], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2]), ([True, 0.5], [2, 3])):
        with pytest.raises(ValueError):
            paged.paged_copy(pool, src, dst)
    i32 = dict(dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        paged.paged_copy(pool, [0], torch.tensor([1], **i32))
    with pytest.raises(TypeError):
        paged.paged_copy(pool, torch.tensor([0], device="cuda"), torch.tensor([1], device="cuda"))
    paged.paged_copy(pool, torch.tensor([0, -1, 9, 1], **i32), torch.tensor([77, 1, 2, -5], **i32))       # no pair names two pages
    paged.paged_copy(pool, [], [])
    paged.paged_copy(pool, torch.tensor([], **i32), torch.tensor([], **i32))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pool, before))


# ----------------------------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("kw", [
    dict(lens=[1]), dict(lens=[1, 2, 15, 16, 17]), dict(lens=[63, 64, 65, 127, 128, 129]), dict(lens=[0, 70, 0, 1]), dict(lens=[0, 0]),
    dict(lens=[300, 5], gs=1), dict(lens=[300, 5], gs=2), dict(lens=[300, 5], gs=3), dict(lens=[300, 5], gs=5, G=1),
    dict(lens=[300, 65], gs=8, G=3), dict(lens=[200], G=8, P=64), dict(lens=[333, 1000], P=128), dict(lens=[100], P=256),
    dict(lens=[260, 31], Rk=8, Rv=8), dict(lens=[260, 31], Rk=24, Rv=40), dict(lens=[260, 31], Rk=40, Rv=72, P=32),
    dict(lens=[260, 31], Rk=48, Rv=128), dict(lens=[260, 31], Rk=96, Rv=136), dict(lens=[260, 31], Rk=128, Rv=384, P=64),
    dict(lens=[260, 31], Rk=136, Rv=256), dict(lens=[260, 31], Rk=192, Rv=264), dict(lens=[260, 31], Rk=256, Rv=512, gs=2),
    dict(lens=[1500, 700], Rk=64, Rv=192, G=8, P=32), dict(lens=[5000], Rk=128, Rv=384, G=1, P=64), dict(lens=[20000], Rk=32, Rv=32, G=1),
    dict(lens=[2100, 64], rotated=True), dict(lens=[777, 3], zeros_int=False), dict(lens=[500], q_std=12.0), dict(lens=[500], q_std=0.01),
    dict(lens=[37 * i % 900 for i in range(70)], G=1, Rk=32, Rv=32)], ids=str)
def test_attention_against_64_bits(kw):
    case = Case(**kw)
    case.check(_run(case))


def test_attention_repeats_bit_for_bit():
    case = Case(lens=[4000, 1, 350, 0, 64], G=4, Rk=128, Rv=384, P=64)
    args = case.args()
    from palu_amd.kernel import paged
    first = paged.paged_attn(*args)
    for _ in range(5):
        assert torch.equal(paged.paged_attn(*args), first)
    case.check(first)


def test_attention_with_unequal_scales():
    """value scales that differ by 2^20 between rows, and one sequence whose weight sits on a row of the smallest scale"""
    case = Case(lens=[400, 130], G=1, Rk=32, Rv=64)
    for b in range(2):
        pages = case.table[b]
        for l in range(case.lens[b]):
            page, off = int(pages[l // case.P]), l % case.P
            old = float(case.vm[page, 0, off, 0])
            new = float(torch.tensor(old * 2.0 ** -(l % 11) * (2.0 ** 9 if l % 3 else 1)).half())
            case.vm[page, 0, off, 0] = new
            case.v[b][0, l] *= new / old
    case.check(_run(case))


def test_a_bad_page_or_length_gives_nan_for_its_sequence_only():
    from palu_amd.kernel import paged
    case = Case(lens=[100, 100, 100, 100], table_pad=0)
    ref, tol = case.reference()
    q, frag, pool, table, lens, qpos = case.args()
    table[1, 3] = case.N                                                       # a page behind the pool
    table[2, 6] = -1
    lens[3] = table.shape[1] * case.P + 1                                      # more rows than the table has pages for
    ctx = paged.paged_attn(q, frag, pool, table, lens, qpos)
    assert ((ctx[0].double() - ref[0]).abs() <= tol[0]).all()
    assert ctx[1:].isnan().all()
    lens[3] = -5                                                               # no rows
    assert (paged.paged_attn(q, frag, pool, table, lens, qpos)[3] == 0).all()


def test_nan_and_infinite_rows_reach_only_their_group():
    case = Case(lens=[90], G=3)
    page = int(case.table[0, 2])
    case.vm[page, 1, 5, 0] = float("inf")
    case.km[page, 2, 5, 0] = float("nan")
    ref, tol = case.reference()
    ctx = _run(case)
    assert ((ctx[0, :4].double() - ref[0, :4]).abs() <= tol[0, :4]).all()
    assert not ctx[0, 4:8].isfinite().any(dim=-1).all() or not ctx[0, 4:8].isfinite().all()
    assert ctx[0, 8:].isnan().all()


def test_strided_queries_tables_and_another_stream():
    from palu_amd.kernel import paged
    case = Case(lens=[210, 33, 0], G=2)
    q, frag, pool, table, lens, qpos = case.args()
    first = paged.paged_attn(q, frag, pool, table, lens, qpos)
    wide = torch.full((3, 2 * case.H + 1, D), 7.0, device="cuda").half()
    wide[:, 1::2] = q
    big = torch.full((3, table.shape[1] + 5), 1 << 20, dtype=torch.int32, device="cuda")
    big[:, :table.shape[1]] = table
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = paged.paged_attn(wide[:, 1::2], frag, pool, big[:, :table.shape[1]], lens, qpos)
        odd = paged.paged_attn(torch.cat((q, q), -1)[:, :, 5:133].roll(5, -1), frag, pool, table, lens, qpos)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, first) and odd.shape == first.shape
    case.check(out)


def test_attention_refuses():
    from palu_amd.kernel import paged
    case = Case(lens=[20])
    q, frag, pool, table, lens, qpos = case.args()
    for args, err in (((q.float(), frag, pool, table, lens), TypeError), ((q[:, :3], frag, pool, table, lens), ValueError),
                      ((q[..., :64], frag, pool, table, lens), ValueError), ((q, frag[:-1], pool, table, lens), ValueError),
                      ((q, frag, pool, table.long(), lens), TypeError), ((q, frag, pool, table, lens.cpu()), ValueError),
                      ((q, frag, pool, table[:0], lens), ValueError), ((q, frag, pool, table, lens, qpos.long()), TypeError),
                      ((q.cpu(), frag, pool, table, lens), TypeError)):
        with pytest.raises(err):
            paged.paged_attn(*args)
    with pytest.raises(ValueError):
        paged.prepare_paged_b(torch.zeros((6, 64, 128), device="cuda").half(), 4)
    with pytest.raises(ValueError):
        paged.prepare_paged_b(torch.zeros((4, 264, 128), device="cuda").half(), 1)
    with pytest.raises(ValueError, match="pick a layer"):
        paged.paged_attn(q, frag, paged.PagePool(*(t[None] for t in pool)), table, lens)
    assert paged.paged_attn(q[:0], frag, pool, table[:0], lens[:0]).shape == (0, case.H, case.Rv)


def test_pages_far_behind_the_start_of_a_large_pool():
    """byte offsets beyond 2^32 in both code arrays"""
    from palu_amd.kernel import paged
    G, P, Rk, Rv = 8, 128, 256, 512
    N = (1 << 32) // (G * P * Rk // 2) + 40
    pool = paged.make_pool(N, G, P, Rk, Rv)                                    # 4.3 GB + 8.6 GB
    case = Case(lens=[300, 129], gs=1, G=G, P=P, Rk=Rk, Rv=Rv)
    far = N - case.N
    for big, small in zip(pool, (case.kc, case.km, case.vc, case.vm)):
        big[far:] = small.cuda()
    q, frag, _, table, lens, qpos = case.args()
    case.check(paged.paged_attn(q, frag, pool, table + far, lens, qpos))
    x, y = torch.randn((1, G, Rk), device="cuda").half(), torch.randn((1, G, Rv), device="cuda").half()
    i = torch.tensor([0], dtype=torch.int32, device="cuda")
    paged.paged_append(pool, x, y, torch.tensor([[N - 1]], dtype=torch.int32, device="cuda"), i, i + 3)
    paged.paged_copy(pool, [N - 1], [1])
    assert torch.equal(pool.v_codes[1].cpu(), pool.v_codes[N - 1].cpu()) and pool.v_codes[1, :, 3].any()
    assert torch.equal(pool.k_meta[1, :, 3].cpu(), pool.k_meta[N - 1, :, 3].cpu())


# ------------------------------------------------------------------------------------------------------- together, as in use
def test_append_fork_and_attend_in_one_captured_graph():
    """A decode step as a server captures it: append the new rows, attend, lengths and tables in buffers the replays read.  Two graphs
    are captured and replayed in turn with eager work between them; every replay equals the eager step."""
    from palu_amd.kernel import paged
    case = Case(lens=[130, 64, 15], G=2, Rk=64, Rv=96, P=16, table_pad=0, spare=6)
    q, frag, pool, table, lens, _ = case.args()
    free = sorted(set(range(case.N)) - set(int(v) for v in case.table.flatten().tolist()))
    full = torch.zeros((3, table.shape[1] + 2), dtype=torch.int32, device="cuda")
    full[:, :table.shape[1]] = table.clamp_min(0)
    for b, n in enumerate(case.lens):                                          # one more page for each sequence
        full[b, (n + case.P - 1) // case.P] = free[b]
    seq = torch.arange(3, dtype=torch.int32, device="cuda")
    k = torch.randn((3, case.G, case.Rk), device="cuda").half()
    v = torch.randn((3, case.G, case.Rv), device="cuda").half()
    pos = lens.clone()

    def step():
        paged.paged_append(pool, k, v, full, seq, pos)
        return paged.paged_attn(q, frag, pool, full, pos + 1, pos)
    eager = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for rep in range(3):
        for gr, out in graphs:
            out.zero_()
            gr.replay()
            assert torch.equal(out, eager)
        k.normal_()
        q.copy_(torch.randn_like(q.float()))
        if rep == 1:
            pos.copy_(pos + 1)
        eager = step().clone()
        torch.cuda.synchronize()


def test_paged_attention_agrees_with_the_single_sequence_path():
    """the same rows in a `QuantLatentCache` and in pages: the decode kernels round keys and weights to fp16 where this path does not,
    so the two agree to those roundings (three of 2^-11 on scores of a few units, and one on the output)"""
    from palu_amd import _lib
    from palu_amd.kernel import paged
    from palu_amd.kernel.abx_rope import prepare_b, rope_inv_freq
    H, G, Rk, Rv, L, P = 32, 8, 128, 384, 1000, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn((L, G, Rk), generator=g, device="cuda").half()
    v = torch.randn((L, G, Rv), generator=g, device="cuda").half()
    b = (torch.randn((H, Rk, D), generator=g, device="cuda") * Rk ** -0.5).half()
    q = torch.randn((H, D), generator=g, device="cuda").half()
    from palu_amd.kernel.palu_attention import QuantLatentCache
    cache = QuantLatentCache(4)
    cache.append_rows(k.transpose(0, 1)[None], v.transpose(0, 1)[None], 0)
    st = cache.buffers(0)
    scores = torch.empty((H, L), dtype=torch.float16, device="cuda")
    inv = rope_inv_freq(k.device)
    _lib.check(_lib.lib.palu_abx_rope_q(q.data_ptr(), D, 1, prepare_b(b, G).data_ptr(), st["kc"].data_ptr(), st["kc"].stride(1),
                                        st["kc"].stride(2), st["km"].data_ptr(), st["km"].stride(1), st["km"].stride(2),
                                        scores.data_ptr(), scores.stride(0), H, G, L, Rk, D, 4, inv.data_ptr(), 0,
                                        _lib.current_stream()))
    from palu_amd.kernel.quant import unpack_dequant
    vd = unpack_dequant(st["vc"][0, :, :L].contiguous(), st["vm"][0, :, :L].contiguous(), 4, Rv)
    p = torch.softmax(scores.float() / math.sqrt(D), -1).view(G, H // G, L)
    want = torch.matmul(p, vd.float()).view(H, Rv)
    pool = paged.make_pool(20, G, P, Rk, Rv)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(2))[:16].to(torch.int32)[None].cuda()
    i = torch.arange(L, dtype=torch.int32, device="cuda")
    paged.paged_append(pool, k, v, table, torch.zeros_like(i), i)
    got = paged.paged_attn(q[None], paged.prepare_paged_b(b, G), pool, table, torch.tensor([L], dtype=torch.int32, device="cuda"))
    torch.testing.assert_close(got[0].float(), want, rtol=2e-3, atol=2e-3)
