"""Modules that decode many sequences on one PagedLatentCache: prompts, forks, steps and compaction together, against a plain
evaluation in 64 bits of the rows that the cache should hold.

The rows themselves are compared bit for bit.  Tolerance of a step's output, beside the module's own roundings of the attention
(fp16, half a step = h = 2^-11): q is rounded to fp16 and the folded query once more, each element by at most h of its value, so a
score, a sum of independent products t, is off with a standard deviation below sqrt(2) h / sqrt(3) * sqrt(sum t^2); six of those are
granted, `d`, with sum t^2 bounded through the absolute values.  The softmax is then off by a factor within exp(+-2 d), its weights
are rounded once more and the context once: e = (exp(2 d) - 1 + h) sum p |v| + h |ctx|.  The output is a sum over contexts in
fp32: |Wo| e, and its rounding, h |out|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D, THETA, h = 128, 10000.0, 2.0 ** -11


def _module(layer, hidden=512, H=8, group_size=4, G=2, rank_k=128, rank_v=128, kv=None, seed=0, theta=THETA, bias=False):
    from palu_amd.kernel.palu_attention import LlamaPaluAttention, build_b

    class Config:
        hidden_size, num_attention_heads, attention_bias = hidden, H, bias
        total_rank_k, total_rank_v, head_dim, num_groups = rank_k, rank_v, D, G
        num_key_value_heads, rope_theta = kv or H, theta
    Config.group_size = group_size
    torch.manual_seed(seed + layer)
    m = LlamaPaluAttention(Config, layer_idx=layer)
    with torch.no_grad():
        for w, fan in ((m.q_proj.weight, hidden), (m.k_proj.VT.weight, hidden), (m.v_proj.VT.weight, hidden),
                       (m.o_proj.weight, m.fused_hidden_dim_o)):
            w.copy_(torch.randn_like(w) * fan ** -0.5)
        m.q_proj.weight.mul_(2)
        m.k_proj.B = torch.nn.Parameter(build_b([u.weight * 0.3 for u in m.k_proj.U_list], group_size, D, m.n_rep))
    return m.half().cuda().eval()


def _dequantise(codes, meta):
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    return (c - meta[..., 1:].double()) * meta[..., :1].double()


def _rows(module, x):
    """The packed rows that the hidden states x [n, hidden] become, [n, G, ..] (k codes, k pairs, v codes, v pairs)"""
    from palu_amd.kernel.quant import quantize_pack
    G = module.num_groups
    return (*quantize_pack(module.k_proj.VT(x).view(len(x), G, -1), 4), *quantize_pack(module.v_proj.VT(x).view(len(x), G, -1), 4))


def _cached(cache, layer, seq):
    n, out = cache.length(seq), []
    for t in cache.pool.layer(layer):
        t = t[cache.pages(seq)].transpose(1, 2)                # [pages, P, G, w]
        out.append(t.reshape(-1, *t.shape[2:])[:n])
    return tuple(out)


def _reference(module, x, rows, pos):
    """One token x [hidden] at position pos over `rows` -> (out, allowed error) in 64 bits"""
    H, gs = module.num_heads, module.group_size
    k, v = _dequantise(*rows[:2]), _dequantise(*rows[2:])      # [n, G, R]
    inv = (1.0 / (module.rope_theta ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D))).double().cuda()

    def turn(t, a):
        return torch.cat((t[..., :64] * a.cos() - t[..., 64:] * a.sin(), t[..., 64:] * a.cos() + t[..., :64] * a.sin()), -1)
    q = module.q_proj.weight.double() @ x.double()
    if module.q_proj.bias is not None:
        q = q + module.q_proj.bias.double()
    q = q.view(H, D)
    rot = turn(q, float(pos) * inv)
    b = module.k_proj.B.double()
    ctx, err = [], []
    for i in range(H):
        key = k[:, i // gs] @ b[i]
        s = turn(key, torch.arange(len(k), device="cuda").double()[:, None] * inv) @ rot[i] / math.sqrt(D)
        p = torch.softmax(s, -1)
        qa, ba = q[i].abs(), b[i].abs()
        f = (qa[:64] * ba[:, :64] + qa[64:] * ba[:, 64:]) ** 2 + (qa[64:] * ba[:, :64] + qa[:64] * ba[:, 64:]) ** 2
        d = 6 * math.sqrt(2 / 3) * h * float((k[:, i // gs] ** 2 @ f.sum(-1)).max().sqrt()) / math.sqrt(D)
        ctx.append(p @ v[:, i // gs])
        err.append((math.exp(2 * d) - 1 + h) * (p @ v[:, i // gs].abs()) + h * ctx[-1].abs())
    w = module.o_proj.weight.double()
    out = w @ torch.cat(ctx)
    tol = w.abs() @ torch.cat(err)
    if module.o_proj.bias is not None:
        out = out + module.o_proj.bias.double()
    return out, tol + h * out.abs() + 2.0 ** -25


def _check(module, x, out, want, pos):
    ref, tol = _reference(module, x, want, pos)
    worst = ((out.double() - ref).abs() / tol).max().item()
    assert worst <= 1.0, worst


def _cat(a, b):
    return tuple(torch.cat(p) for p in zip(a, b))


@torch.no_grad()
@pytest.mark.parametrize("P,kw", [(16, {}), (64, dict(kv=4, group_size=2, rank_k=96, rank_v=192, theta=5e5)),
                                  (32, dict(H=6, group_size=3, rank_k=512, rank_v=768, bias=True))])
def test_prompts_forks_steps_and_compaction_together(P, kw):
    """Two layers; prompts of odd lengths, forks that share an open page, sequences that come and end, a compaction and a smaller
    pool in between.  Every cached row is the quantised row of its token, every output the attention over exactly those rows."""
    from palu_amd.kernel.palu_attention import PagedLatentCache, QuantLatentCache
    mods = [_module(i, **kw) for i in range(2)]
    m0 = mods[0]
    cache = PagedLatentCache(2, m0.num_groups, m0.group_rank_k, m0.group_rank_v, num_pages=40, max_seqs=5, max_pages=12, page_size=P)
    g = torch.Generator().manual_seed(P)
    rows = {}                                                  # (sequence, layer) -> packed rows

    def prompt(ids, n):
        x = torch.randn((len(ids), n, 512), generator=g).half().cuda()
        cache.begin(ids, tokens=n)
        for li, m in enumerate(mods):
            out, probs, back = m(x, past_key_value=cache, is_causal=True)
            assert out.shape == x.shape and probs is None and back is cache
            for j, i in enumerate(ids):
                one = QuantLatentCache(4)
                same = m(x[j:j + 1], past_key_value=one, is_causal=True)[0]
                assert torch.equal(out[j:j + 1], same)
                st = one.buffers(li)
                rows[i, li] = tuple(st[k][0, :, :n].transpose(0, 1) for k in ("kc", "km", "vc", "vm"))
        cache.commit()

    def step(ids):
        x = torch.randn((len(ids), 1, 512), generator=g).half().cuda()
        cache.begin(ids)
        outs = [m(x, past_key_value=cache)[0] for m in mods]
        cache.commit()
        for li, m in enumerate(mods):
            new = _rows(m, x[:, 0])
            for j, i in enumerate(ids):
                rows[i, li] = _cat(rows[i, li], tuple(t[j:j + 1] for t in new)) if (i, li) in rows else tuple(t[j:j + 1] for t in new)
                _check(m, x[j, 0], outs[li][j, 0], rows[i, li], cache.length(i) - 1)

    def same_rows():
        for i in cache.sequences:
            for li in range(2):
                if (i, li) in rows:
                    assert all(torch.equal(a, b) for a, b in zip(_cached(cache, li, i), rows[i, li])), (i, li)

    a, b = cache.add(), cache.add()
    prompt([a], P + 5)
    prompt([b], 2 * P)
    c = cache.add()
    prompt([c], 7)
    d = cache.fork(a)
    rows.update({(d, li): rows[a, li] for li in range(2)})
    step([d, b, a])                                            # d copies the page that it shares with a
    same_rows()
    e = cache.add()
    step([e, a])                                               # a first token without a prompt
    step([c])
    cache.free(b)
    assert cache.compact() == 40 - cache.num_free
    cache.resize(20)
    same_rows()
    for _ in range(3):
        step([a, c, d, e])
    same_rows()


@torch.no_grad()
def test_a_captured_step_serves_later_steps():
    """The kernels of a decode step read its lengths, positions and table from the device: one capture, many steps (with a page
    boundary, a fork and a compaction between them), each against the same step run eagerly on a copy of the cache."""
    import copy

    from palu_amd.kernel.palu_attention import PagedLatentCache
    m = _module(0).prepare_decode(paged=True)
    cache = PagedLatentCache(1, m.num_groups, m.group_rank_k, m.group_rank_v, num_pages=40, max_seqs=3, max_pages=8, page_size=16)
    g = torch.Generator().manual_seed(3)
    a, b, dead = cache.add(), cache.add(), cache.add()
    for i, n in ((dead, 20), (a, 30), (b, 3)):
        cache.begin([i], tokens=n)
        m(torch.randn((1, n, 512), generator=g).half().cuda(), past_key_value=cache, is_causal=True)
        cache.commit()
    x = torch.randn((2, 1, 512), generator=g).half().cuda()
    cache.begin([a, b])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m(x, past_key_value=cache)                             # warm-up; the captured step writes the same rows again
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m(x, past_key_value=cache)[0]
    graph.replay()
    cache.commit()
    for i in range(6):
        if i == 2:
            cache.free(dead)
            cache.compact()
        if i == 4:
            cache.fork(a)
        x.copy_(torch.randn((2, 1, 512), generator=g).half())
        ids = [b, a] if i == 5 else [a, b]
        cache.begin(ids)
        twin = copy.copy(cache)
        twin._layers = [type(cache.pool)(*(t[0].clone() for t in cache.pool))]
        want = m(x, past_key_value=twin)[0]
        torch.cuda.synchronize()
        graph.replay()
        cache.commit()
        assert torch.equal(out, want)
        for p, q in zip(cache.pool, twin._layers[0]):
            assert torch.equal(p[0], q)


@torch.no_grad()
def test_the_weights_layout_follows_the_weight():
    """the layout of B is kept per weight: load_state_dict, and a write that is announced, make a new one; a capture makes none"""
    from palu_amd.kernel.abx_rope import invalidate_b, paged_b
    from palu_amd.kernel.paged import prepare_paged_b
    m = _module(0)
    first = paged_b(m.k_proj.B, 2)
    assert paged_b(m.k_proj.B, 2) is first
    state = {k: v * 2 for k, v in m.k_proj.state_dict().items()}
    m.k_proj.load_state_dict(state)
    second = paged_b(m.k_proj.B, 2)
    assert not torch.equal(first, second) and torch.equal(second, prepare_paged_b(m.k_proj.B.detach(), 2))
    m.k_proj.B.data.mul_(2)
    invalidate_b(m.k_proj.B)
    assert torch.equal(paged_b(m.k_proj.B, 2), prepare_paged_b(m.k_proj.B.detach(), 2))


@torch.no_grad()
def test_module_refusals_on_the_gpu():
    from palu_amd.kernel.palu_attention import PagedLatentCache
    m = _module(0)
    cache = PagedLatentCache(1, 2, 64, 64, num_pages=8, max_seqs=2, max_pages=4, page_size=16)
    a, b = cache.add(), cache.add()
    x = torch.randn(2, 5, 512).half().cuda()
    cache.begin([a, b], tokens=5)
    causal = torch.full((5, 5), float("-inf")).triu(1).half().cuda()
    with pytest.raises(ValueError, match="causal mask only"):
        m(x, attention_mask=torch.zeros(2, 1, 5, 5).half().cuda(), past_key_value=cache)
    with pytest.raises(ValueError, match="Attention mask should be"):
        m(x, attention_mask=torch.zeros(2, 1, 5, 6).half().cuda(), past_key_value=cache)
    with pytest.raises(ValueError, match="positions 0"):
        m(x, position_ids=torch.arange(1, 6).cuda()[None], past_key_value=cache)
    out = m(x, attention_mask=causal.expand(2, 1, 5, 5), past_key_value=cache)[0]
    assert torch.equal(out, m(x, past_key_value=cache, is_causal=True)[0])
    assert torch.equal(out, m(x, attention_mask=causal[None, None] == 0, position_ids=torch.arange(5).cuda()[None], past_key_value=cache)[0])
    cache.commit()
    cache.begin([a, b], tokens=2)
    with pytest.raises(NotImplementedError, match="starts an empty sequence"):
        m(x[:, :2], past_key_value=cache)
    cache.abort()
    cache.begin([a, b])
    with pytest.raises(ValueError, match="no attention mask"):
        m(x[:, :1], attention_mask=causal.new_zeros(2, 1, 1, 6), past_key_value=cache)
    own = m(x[:, :1], past_key_value=cache)[0]
    assert torch.equal(own, m(x[:, :1], position_ids=torch.tensor([[5], [5]]).cuda(), past_key_value=cache)[0])
    assert torch.equal(own, m(x[:, :1], position_ids=torch.tensor([[5]]).cuda(), past_key_value=cache)[0])
    with pytest.raises(ValueError, match="is not empty"):
        cache.adopt(0, None)


@torch.no_grad()
def test_the_registered_ops_are_the_same_kernels():
    from palu_amd import ops  # noqa: F401
    from palu_amd.kernel import paged
    from palu_amd.kernel.quant import quantize_pack
    g = torch.Generator().manual_seed(9)
    pool = paged.make_pool(6, 2, 16, 64, 96)
    table = torch.tensor([[4, 1], [0, 3]], dtype=torch.int32).cuda()
    k, v = (torch.randn((40, 2, r), generator=g).half().cuda() for r in (64, 96))
    seq = torch.tensor([0] * 23 + [1] * 17, dtype=torch.int32).cuda()
    pos = torch.tensor([*range(23), *range(17)], dtype=torch.int32).cuda()
    torch.ops.palu.paged_append(*pool, k, v, table, seq, pos)
    codes, meta = quantize_pack(k[16:23], 4)
    assert torch.equal(pool.k_codes[1, :, :7].transpose(0, 1), codes) and torch.equal(pool.k_meta[1, :, :7].transpose(0, 1), meta)
    pair = torch.tensor([[1], [5]], dtype=torch.int32).cuda()
    torch.ops.palu.paged_copy(*pool, pair[0], pair[1])
    assert all(torch.equal(t[1], t[5]) for t in pool)
    q = torch.randn((2, 8, D), generator=g).half().cuda()
    frag = paged.prepare_paged_b(torch.randn((8, 64, D), generator=g).half().cuda() * 0.1, 2)
    lens = torch.tensor([23, 17], dtype=torch.int32).cuda()
    one = torch.ops.palu.paged_attn(q, frag, *pool, table, lens, lens - 1, THETA)
    assert torch.equal(one, paged.paged_attn(q, frag, pool, table, lens, lens - 1, THETA))
    moved = table.clone()
    moved[0, 1] = 5
    assert torch.equal(one, paged.paged_attn(q, frag, pool, moved, lens, lens - 1, THETA))
    with torch._subclasses.FakeTensorMode(allow_non_fake_inputs=True):
        assert torch.ops.palu.paged_attn(q, frag, *pool, table, lens).shape == (2, 8, 96)


@torch.no_grad()
def test_a_step_does_not_begin_inside_a_capture():
    from palu_amd.kernel.palu_attention import PagedLatentCache
    cache = PagedLatentCache(1, 2, 64, 64, num_pages=8, max_seqs=2, max_pages=4, page_size=16)
    a = cache.add()
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with pytest.raises(RuntimeError, match="not inside a graph capture"):
            cache.begin([a])
    cache.begin([a])
    cache.abort()
    assert cache.num_free == 7


@torch.no_grad()
def test_two_streams_work_on_two_caches_at_once():
    """the same module, two caches, two streams: nothing of a call is shared but the weights"""
    from palu_amd.kernel.palu_attention import PagedLatentCache
    m = _module(0).prepare_decode(paged=True)
    g = torch.Generator().manual_seed(5)
    xs = [torch.randn((3, 1, 512), generator=g).half().cuda() for _ in range(2)]
    prompts = [torch.randn((3, n, 512), generator=g).half().cuda() for n in (200, 333)]

    def run(i):
        cache = PagedLatentCache(1, 2, 64, 64, num_pages=80, max_seqs=3, max_pages=24, page_size=16)
        ids = [cache.add() for _ in range(3)]
        cache.begin(ids, tokens=prompts[i].shape[1])
        m(prompts[i], past_key_value=cache, is_causal=True)
        cache.commit()
        outs = []
        for _ in range(20):
            cache.begin(ids)
            outs.append(m(xs[i], past_key_value=cache)[0])
            cache.commit()
        return torch.cat(outs)
    want = [run(0), run(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(run(i))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
