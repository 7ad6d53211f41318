"""apply_rotary, norm_rotary and append_kvcache on the GPU against the 64-bit oracle.

Tolerance of an element y: half a step of its type, eps / 2 |y| (fp16: or half its smallest subnormal, 2^-25), for the
one rounding, and for the fp32 arithmetic before it 2^-19 of the magnitudes that went into it: the table's and the
products' roundings are 4 x 2^-24 of those, and a norm's sum of up to 64 squares a lane and its scale, weight and
reciprocal root under 2^-20 more.
"""

import math

import pytest
import torch

import lvattn
from oracle import rotary as R

pytestmark = pytest.mark.gpu
EPS = 1e-6


def close(got, want, size):
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() + 2.0 ** -19 * size
    if got.dtype == torch.float16:
        tol += 2.0 ** -25
    bad = (got.cpu().double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def draw(t, heads, dim, dtype, seed, pad=0):
    """Views [T, H, dim] of one [T, sum(heads) dim + pad] projection on the CPU; pad % 8 != 0 misaligns the tokens."""
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(t, sum(heads) * dim + pad, generator=gen) * 2).to(dtype)
    return x, [y.view(t, -1, dim) for y in x[:, :sum(heads) * dim].split([h * dim for h in heads], 1)]


def views(x, heads, dim, cuda):
    x = x.to(cuda)
    return [y.view(x.size(0), -1, dim) for y in x[:, :sum(heads) * dim].split([h * dim for h in heads], 1)]


CASES = [  # tokens, heads, kv heads, dim, rotary dim, pad
    (1, 16, 8, 128, 128, 0), (3, 32, 8, 128, 128, 0), (257, 40, 8, 64, 64, 0), (65, 7, 1, 128, 64, 0),
    (33, 8, 8, 256, 64, 0), (18, 5, 3, 96, 96, 0), (70, 16, 2, 80, 80, 8), (19, 16, 2, 80, 32, 0), (5, 4, 2, 192, 192, 0),
    (9, 3, 1, 512, 512, 0), (7, 2, 1, 576, 64, 0), (6, 2, 1, 1024, 128, 0),
    (21, 5, 1, 128, 128, 1), (11, 3, 2, 80, 20, 0), (8, 2, 2, 6, 4, 0), (130, 1, 1, 2, 2, 0), (2, 3, 1, 130, 66, 3),
    (900, 2, 1, 64, 16, 4), (13, 5, 2, 96, 24, 0), (9, 6, 2, 64, 20, 0), (5, 2, 1, 256, 40, 0), (4, 2, 1, 512, 18, 0),
    (3, 2, 1, 1024, 100, 0),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,hq,hk,dim,rot,pad", CASES)
def test_rotary_and_norm_match_the_oracle(cuda, t, hq, hk, dim, rot, pad, dtype, interleaved):
    scaling = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096) if rot > 20 else None
    base, most = 10000.0, 20000
    gen = torch.Generator().manual_seed(t)
    positions = torch.randint(0, most, (t,), generator=gen)
    positions[-1] = most - 1
    x, (q, k) = draw(t, (hq, hk), dim, dtype, 10 * t + dim, pad)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype) for _ in range(2))
    table = lvattn.rotary_table(rot, most, base, scaling, device=cuda)
    dq, dk = views(x, (hq, hk), dim, cuda)
    kw = dict(base=base, scaling=scaling, interleaved=interleaved)
    got = lvattn.apply_rotary(dq, dk, positions.to(cuda), table, interleaved=interleaved)
    for y, z in zip(got, (q, k)):
        assert y.is_contiguous()
        close(y, *R.rotate(z, positions, rot, **kw))
    got = lvattn.norm_rotary(dq, dk, wq.to(cuda), wk.to(cuda), positions.to(cuda), table, EPS, interleaved)
    for y, z, w in zip(got, (q, k), (wq, wk)):
        close(y, *R.rotate(z, positions, rot, weight=w, eps=EPS, **kw))
    # In place, one of the two normed, the same bits; the padding behind the heads stays.
    kept = x[:, (hq + hk) * dim:]
    in_place = x.to(cuda)
    iq, ik = (y.view(t, -1, dim) for y in in_place[:, :(hq + hk) * dim].split([hq * dim, hk * dim], 1))
    lvattn.norm_rotary(iq, ik, wq.to(cuda), None, positions.to(cuda), table, EPS, interleaved, out_q=iq, out_k=ik)
    plain_k = lvattn.apply_rotary(None, dk, positions.to(cuda), table, interleaved=interleaved)
    assert plain_k[0] is None and torch.equal(iq, got[0]) and torch.equal(ik, plain_k[1])
    assert torch.equal(in_place[:, (hq + hk) * dim:].cpu(), kept)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_call_larger_than_the_cache_gives_the_bits_of_its_parts(cuda, dim, dtype, interleaved):
    """Past 128 MB read and written the chunks go past the caches: the same bits as token ranges on their own."""
    hq, hk, bs = 4, 2, 32
    t = (130 << 20) // ((hq + 2 * hk) * dim * 4)
    gen = torch.Generator(device=cuda).manual_seed(dim)
    x = torch.randn(t, (hq + 2 * hk) * dim, device=cuda, generator=gen).to(dtype)
    q, k, v = (y.view(t, -1, dim) for y in x.split([hq * dim, hk * dim, hk * dim], 1))
    pos = torch.randint(0, 5000, (t,), device=cuda, generator=gen)
    slots = torch.randperm((t // bs + 2) * bs, device=cuda, generator=gen)[:t].int()
    w, table = torch.randn(dim, device=cuda, generator=gen).to(dtype), lvattn.rotary_table(dim, 5000, device=cuda)
    backend = lvattn.MI355XAttention(hq, dim, 1.0, hk)
    runs = []
    for step in (t, t // 3 + 1):
        caches = [torch.zeros(t // bs + 2, bs, hk, dim, dtype=dtype, device=cuda) for _ in range(2)]
        outs = [backend.append_kvcache(q[a:a + step], k[a:a + step], v[a:a + step], *caches, slots[a:a + step],
                                       pos[a:a + step], table, q_weight=w, k_weight=w, interleaved=interleaved)
                for a in range(0, t, step)]
        runs.append((torch.cat(outs), *caches))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    close(runs[0][0][-2:], *R.rotate(q[-2:].cpu(), pos[-2:].cpu(), dim, weight=w.cpu(), eps=EPS,
                                        interleaved=interleaved))


def test_odd_positions(cuda):
    """Padding rows' negative positions rotate as position 0, one past the table gives NaN in the rotated dims alone."""
    for dim, rot in ((128, 64), (80, 20)):
        q = torch.randn(4, 3, dim, device=cuda).to(torch.bfloat16)
        table = lvattn.rotary_table(rot, 100, device=cuda)
        positions = torch.tensor([-1, 100, 99, 1 << 40], device=cuda)
        y, _ = lvattn.apply_rotary(q, None, positions, table)
        assert torch.equal(y[0], q[0]) and torch.equal(y[:, :, rot:], q[:, :, rot:])
        assert y[[1, 3], :, :rot].isnan().all() and y[2].isfinite().all()


def test_views_of_part_of_a_head_in_place(cuda):
    """Latent attention's rope dims: the last 64 of 192-wide query heads and of 576-wide latents, in place, interleaved; the
    other dims stay."""
    q, latent = (torch.randn(9, *shape, device=cuda).to(torch.bfloat16) for shape in ((16, 192), (576,)))
    table, pos = lvattn.rotary_table(64, 500, device=cuda), torch.arange(9, device=cuda) * 50
    want_q, want_l = q.clone(), latent.clone()
    rope = [q[..., 128:], latent[:, None, 512:]]
    lvattn.apply_rotary(*rope, pos, table, interleaved=True, out_q=rope[0], out_k=rope[1])
    for got, x, n in ((q, want_q, 128), (latent[:, None], want_l[:, None], 512)):
        assert torch.equal(got[..., :n], x[..., :n])
        close(got[..., n:], *R.rotate(x[..., n:].cpu(), pos.cpu(), 64, interleaved=True))


def test_not_a_number_stays_in_its_head(cuda):
    q = torch.randn(6, 8, 128, device=cuda).to(torch.bfloat16)
    w, table = torch.ones(128, device=cuda, dtype=torch.bfloat16), lvattn.rotary_table(128, 10, device=cuda)
    pos = torch.arange(6, device=cuda)
    want, _ = lvattn.norm_rotary(q, None, w, None, pos, table)
    bad = q.clone()
    bad[2, 3, 5], bad[4, 7, 127] = math.nan, math.inf
    got, _ = lvattn.norm_rotary(bad, None, w, None, pos, table)
    touched = torch.zeros(6, 8, dtype=torch.bool, device=cuda)
    touched[2, 3] = touched[4, 7] = True
    assert torch.equal(got[~touched], want[~touched]) and got[2, 3].isnan().all()
    assert got[4, 7].isnan().any()  # inf * 0, as the formula has it
    zeros, _ = lvattn.norm_rotary(torch.zeros_like(q), None, w, None, pos, table)
    assert not zeros.any()


def test_no_tokens(cuda):
    q, table = torch.empty(0, 4, 64, device=cuda, dtype=torch.float16), lvattn.rotary_table(64, 8, device=cuda)
    pos = torch.empty(0, dtype=torch.int64, device=cuda)
    assert lvattn.apply_rotary(q, q, pos, table)[0].shape == (0, 4, 64)
    cache = torch.ones(2, 16, 4, 64, device=cuda, dtype=torch.float16)
    out = lvattn.MI355XAttention(4, 64, 1.0, 4).append_kvcache(q, q, q, cache, cache.clone(), pos.int(), pos, table)
    assert out.shape == (0, 4, 64) and (cache == 1).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("t,hq,hk,dim,rot,pad,bs", [
    (1, 16, 8, 128, 128, 0, 16), (3, 32, 8, 128, 128, 0, 256), (200, 8, 2, 64, 64, 0, 16), (37, 7, 1, 64, 32, 0, 48),
    (61, 4, 2, 80, 20, 0, 16), (45, 3, 3, 128, 128, 1, 7), (10, 2, 2, 256, 256, 0, 16), (513, 1, 1, 128, 96, 0, 64)])
def test_append_matches_rotary_and_store(cuda, t, hq, hk, dim, rot, pad, bs, normed, layout, interleaved):
    """The queries against the oracle; the caches hold the rotated keys (the bits of norm_rotary) and the values where a
    slot names them, and what they held before everywhere else."""
    dtype, blocks, most = torch.bfloat16, t // bs + 3, 4096
    heads = (hq, hk, hk)
    gen = torch.Generator().manual_seed(dim + t)
    x, (q, k, v) = draw(t, heads, dim, dtype, t, pad)
    positions = torch.randint(0, most, (t,), generator=gen)
    slots = torch.randperm(blocks * bs, generator=gen)[:t].to(torch.int32)
    slots[torch.randperm(t, generator=gen)[:t // 5]] = -1
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype) if normed else None for _ in range(2))
    shape = (blocks, bs, hk, dim) if layout == "NHD" else (blocks, hk, bs, dim)
    caches = [torch.randn(shape, generator=gen).to(dtype).to(cuda) for _ in range(2)]
    if layout == "HND":
        caches = [c.transpose(1, 2) for c in caches]
    table = lvattn.rotary_table(rot, most, device=cuda)
    dq, dk, dv = views(x, heads, dim, cuda)
    want = [c.clone() for c in caches]
    backend = lvattn.MI355XAttention(hq, dim, 1.0, hk)
    dw = [None if w is None else w.to(cuda) for w in (wq, wk)]
    got = backend.append_kvcache(dq, dk, dv, *caches, slots.to(cuda), positions.to(cuda), table, q_weight=dw[0],
                                 k_weight=dw[1], eps=EPS, interleaved=interleaved)
    close(got, *R.rotate(q, positions, rot, interleaved=interleaved, weight=wq, eps=EPS))
    _, turned = lvattn.norm_rotary(None, dk, None, dw[1], positions.to(cuda), table, EPS, interleaved)
    close(turned, *R.rotate(k, positions, rot, interleaved=interleaved, weight=wk, eps=EPS))
    kept = slots >= 0
    page, at = (slots[kept] // bs).long().to(cuda), (slots[kept] % bs).long().to(cuda)
    want[0][page, at], want[1][page, at] = turned[kept.to(cuda)], dv[kept.to(cuda)]
    assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])
    # Only the keys and values (no queries), int64 slots, into the same places: the caches stay as they are.
    assert backend.append_kvcache(None, dk, dv, *caches, slots.long().to(cuda), positions.to(cuda), table,
                                  k_weight=dw[1], eps=EPS, interleaved=interleaved) is None
    assert torch.equal(caches[0], want[0]) and torch.equal(caches[1], want[1])


def test_append_past_32_bit_offsets(cuda):
    """A cache of more than 2^32 bytes: slots at its end land there (NHD, and HND strides)."""
    hk, dim, bs, blocks = 8, 128, 16, 140_000  # 4.6 GB a cache
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, hk, dim, generator=gen).to(torch.bfloat16).to(cuda) for _ in range(2))
    k_cache, v_cache = (torch.empty(blocks, bs, hk, dim, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    slots = torch.tensor([blocks * bs - 1, 5, blocks * bs - 17], dtype=torch.int32, device=cuda)
    pos, table = torch.zeros(3, dtype=torch.int64, device=cuda), lvattn.rotary_table(128, 4, device=cuda)
    lvattn.MI355XAttention(hk, dim, 1.0, hk).append_kvcache(None, k, v, k_cache, v_cache, slots, pos, table)
    for i, s in enumerate(slots.tolist()):
        assert torch.equal(k_cache[s // bs, s % bs], k[i]) and torch.equal(v_cache[s // bs, s % bs], v[i])


def test_append_replays_in_a_graph_and_on_another_stream(cuda):
    t, hq, hk, dim, bs = 24, 8, 2, 128, 16
    x, _ = draw(t, (hq, hk, hk), dim, torch.bfloat16, 3)
    xs = [x.to(cuda), draw(t, (hq, hk, hk), dim, torch.bfloat16, 4)[0].to(cuda)]
    static = xs[0].clone()
    q, k, v = (y.view(t, -1, dim) for y in static.split([hq * dim, hk * dim, hk * dim], 1))
    caches = [torch.zeros(4, bs, hk, dim, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    slots, pos = torch.arange(t, dtype=torch.int32, device=cuda), torch.arange(t, device=cuda)
    table, backend = lvattn.rotary_table(dim, 64, device=cuda), lvattn.MI355XAttention(hq, dim, 1.0, hk)
    out = backend.append_kvcache(q, k, v, *caches, slots, pos, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backend.append_kvcache(q, k, v, *caches, slots, pos, table, out=out)
    side = torch.cuda.Stream()
    for i in range(4):
        static.copy_(xs[i % 2])
        pos.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.zeros_like(c) for c in caches]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = backend.append_kvcache(q, k, v, *eager, slots, pos, table)
        side.synchronize()
        assert torch.equal(out, again) and all(torch.equal(a, b) for a, b in zip(caches, eager))


@pytest.mark.parametrize("query_len", [1, 3], ids=["decode", "drafts"])
def test_decode_graphs_rotate_inside(cuda, query_len):
    """DecodeGraphs with a rotary table: a replay of raw projections equals rotating them into the cache and attending
    eagerly, bit for bit in the cache and the queries' attention, with padding rows that store nothing."""
    hq, hk, dim, bs, blocks, most = 8, 2, 128, 16, 48, 6
    backend, dt = lvattn.MI355XAttention(hq, dim, 0.09, hk), torch.bfloat16
    gen = torch.Generator().manual_seed(query_len)
    caches = [torch.randn(blocks, bs, hk, dim, generator=gen).to(dt).to(cuda) for _ in range(2)]
    w = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dt).to(cuda)
    rotary = dict(table=lvattn.rotary_table(dim, 256, device=cuda), q_weight=w, k_weight=w, eps=1e-5)
    graphs = lvattn.DecodeGraphs(backend, *caches, [4, 8], most, query_len, rotary=rotary)
    before = [c.clone() for c in caches]
    graphs.capture()
    assert all(torch.equal(a, b) for a, b in zip(caches, before))  # padding rows only
    packer = lvattn.Packer(cuda, bs)
    for turn, rows in enumerate((3, 8, 1, 4)):
        pages = torch.randperm(blocks, generator=gen)[:rows * most].view(rows, most).tolist()
        cached = torch.randint(0, most * bs - query_len + 1, (rows,), generator=gen).tolist()
        lists = [p[:-(-(c + query_len) // bs)] for p, c in zip(pages, cached)]
        t = rows * query_len
        q, k, v = (torch.randn(t, h, dim, generator=gen).to(dt).to(cuda) for h in (hq, hk, hk))
        eager = [c.clone() for c in caches]
        got = graphs.replay(cached, lists, q, k, v).clone()
        positions, fields = packer.pack(cached, [query_len] * rows, lists, num_speculative_tokens=query_len - 1,
                                        is_prompt=[False] * rows)
        fields.pop("order")
        ctx = lvattn.Context(**fields)
        turned = backend.append_kvcache(q, k, v, *eager, ctx.slot_mapping, positions, **rotary)
        assert all(torch.equal(a, b) for a, b in zip(caches, eager))
        y, size = R.rotate(q.cpu(), positions.cpu(), dim, weight=w.cpu(), eps=1e-5)
        close(turned, y, size)
        want = backend.forward(turned, k, v, *eager, ctx)
        # the graph's bound on the keys may split them otherwise: the outputs' own tolerance in this repository
        torch.testing.assert_close(got.float(), want.float(), atol=2e-2, rtol=1e-2)
