"""decode_shared on the GPU against attention in 64 bits, row by row.

Tolerance of an element y = sum p v / sum p, with A = sum p |v| / sum p: half a step of its type, h = eps / 2, relative to y
for the output's rounding; h A for the probabilities, each rounded once to the same type before P V; and for the fp32
arithmetic 2^-12 A: a score of D products errs by at most D 2^-24 of the magnitudes that it sums (about 11 at D = 128 and
the sizes drawn here, so 2^-13.5), which is the relative error of a probability and again of their sum, and sums of some
thousand terms and the merges stay below 2^-14. (fp16: and half its smallest subnormal, 2^-25.) Where keys are scaled up,
`score` is that error of p and of its sum, 2 D 2^-24 max sum |q k| scale, in the place of the 2^-13.5's.
"""

import math

import pytest
import torch

from lvattn import Context, DecodeGraphs, MI355XAttention, Packer, apply_rotary, rotary_table, shared_prefix_len

pytestmark = pytest.mark.gpu


def step(shared, owns, *, hq, hk, dim, page, dtype, layout="NHD", queries=1, seed=0, spare=3, extra_width=0, fill=math.nan):
    """Caches (`fill` wherever no row's keys lie), whole tables, lengths and queries of rows that share `shared` keys and
    have owns[i] more (None: a padding row of no keys)."""
    gen = torch.Generator().manual_seed(seed)
    tails = [0 if n is None else -(-n // page) for n in owns]
    head, width = shared // page, shared // page + max(tails) + extra_width
    blocks = head + sum(tails) + spare
    perm = torch.randperm(blocks, generator=gen)
    k = torch.full((blocks, page, hk, dim), fill, dtype=dtype)
    v = torch.full((blocks, page, hk, dim), fill, dtype=dtype)
    tables = torch.full((len(owns), max(width, 1)), -1, dtype=torch.int32)
    at = head

    def put(blk, n):
        for c in (k, v):
            c[blk, :n] = torch.randn(n, hk, dim, generator=gen).to(dtype)

    for b in perm[:head]:
        put(b, page)
    for i, (n, t) in enumerate(zip(owns, tails)):
        if n is None:
            continue
        tables[i, :head] = perm[:head]
        tables[i, head:head + t] = perm[at:at + t]
        for j in range(t):
            put(perm[at + j], min(page, n - j * page))
        at += t
    lens = torch.tensor([0 if n is None else shared + n for n in owns], dtype=torch.int32)
    q = (torch.randn(len(owns) * queries, hq, dim, generator=gen) * 1.5).to(dtype)
    if layout == "HND":
        k, v = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (k, v))
    return q, k, v, tables, lens


def on(device, x):  # keeps a transposed view's strides
    return x.to(device) if x.is_contiguous() else x.transpose(1, 2).to(device).transpose(1, 2)


def want(q, k, v, tables, lens, queries, scale, rows=None):
    """(y, A) of the rows, in 64 bits."""
    page, hk, dim = k.shape[1:]
    hq = q.size(1)
    y, a = (torch.zeros(q.shape, dtype=torch.float64) for _ in range(2))
    for i in range(lens.numel()) if rows is None else rows:
        n = int(lens[i])
        if n == 0:
            continue
        pages = tables[i, :-(-n // page)].long()
        ks, vs = (c[pages].reshape(-1, hk, dim)[:n].double().repeat_interleave(hq // hk, 1) for c in (k, v))
        for j in range(queries):
            sees = n - queries + j + 1
            if sees <= 0:
                continue
            t = i * queries + j
            p = (torch.einsum("hd,khd->hk", q[t].double(), ks[:sees]) * scale).softmax(-1)
            y[t], a[t] = torch.einsum("hk,khd->hd", p, vs[:sees]), torch.einsum("hk,khd->hd", p, vs[:sees].abs())
    return y, a


def close(got, y, a, rows=slice(None), score=0.0):
    got, y, a = got.cpu()[rows], y[rows], a[rows]
    h = torch.finfo(got.dtype).eps / 2
    tol = h * y.abs() + (h + 2.0 ** -12 + score) * a + (2.0 ** -25 if got.dtype == torch.float16 else 0)
    bad = ~((got.double() - y).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}"


def attend(cuda, shared, q, k, v, tables, lens, scale, out=None):
    hq, hk, dim = q.size(1), k.size(2), q.size(2)
    ctx = Context(context_lens=lens.to(cuda), block_tables=tables.to(cuda))
    return MI355XAttention(hq, dim, scale, hk).decode_shared(q.to(cuda), on(cuda, k), on(cuda, v), ctx, shared, out=out)


CASES = [  # shared, own keys, queries, hq, hk, dim, page
    (2048, [1, 300, 17, 64], 1, 16, 8, 128, 16),
    (256, [40], 1, 8, 2, 64, 16),
    (512, [1, 2, 63, 64, 65, 16, 15, 0], 1, 32, 8, 128, 32),
    (768, [5] * 40, 1, 32, 8, 128, 256),
    (64, [100, 33], 3, 16, 2, 64, 64),
    (1024, [7, 90, 3, 200, 31, 33, 90], 5, 28, 4, 128, 64),
    (480, [10, 47, 48, 49, 300], 2, 10, 2, 128, 48),
    (160, [1, 81, 79], 1, 7, 1, 64, 80),
    (0, [1, 400, 31], 1, 8, 4, 128, 16),
    (16, [1, 1], 1, 4, 4, 128, 16),
    (4096, [20, 700, 1], 1, 64, 1, 64, 16),
    (1536, [33, 1000], 1, 64, 1, 128, 128),
    (960, [9] * 130, 1, 24, 8, 64, 64),
    (1280, [2, 3] * 50, 2, 40, 8, 128, 256),
    (8192, [600, 5, 1200], 1, 16, 8, 64, 16),
    (192, [4] * 300, 1, 16, 2, 128, 48),
]


@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shared,owns,queries,hq,hk,dim,page", CASES)
def test_matches_attention_row_by_row(cuda, shared, owns, queries, hq, hk, dim, page, dtype, layout):
    s = step(shared, owns, hq=hq, hk=hk, dim=dim, page=page, dtype=dtype, layout=layout, queries=queries,
             seed=shared + len(owns))
    scale = dim ** -0.5
    close(attend(cuda, shared, *s, scale), *want(*s, queries, scale))


# The kernels of a call: how the prefix is computed (few-query items of 16, 32 or 64 rows, or prompt items on pages of
# 64, 32 or 16), and the rows' own keys (16, 32 or 64 rows, or 16 of a pair of kv heads). rows, queries, hq, hk, page.
KERNELS = {
    "few16-16": (4, 1, 8, 4, 64), "few16-pairs": (8, 1, 32, 32, 16), "few32-16": (10, 1, 8, 4, 32),
    "few32-32": (1, 3, 16, 2, 16), "few32-pairs": (16, 1, 32, 16, 64), "few64-16": (40, 1, 2, 1, 48),
    "few64-pairs": (40, 1, 16, 8, 48), "few64-32": (5, 3, 8, 1, 48), "few64-64": (5, 5, 16, 2, 48),
    **{f"tile{page}-{own}": (*shape, page) for page in (64, 32, 16) for own, shape in
       {"16": (40, 1, 2, 1), "pairs": (40, 1, 16, 8), "32": (5, 3, 8, 1), "64": (5, 5, 16, 2)}.items()}}


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", KERNELS)
def test_every_kernel(cuda, name, dtype, dim):
    rows, queries, hq, hk, page = KERNELS[name]
    owns = [queries + (37 * i) % 70 for i in range(rows)]
    owns[-1] = 530  # two splits of a row's own keys
    s = step(576, owns, hq=hq, hk=hk, dim=dim, page=page, dtype=dtype, queries=queries, seed=rows)
    close(attend(cuda, 576, *s, dim ** -0.5), *want(*s, queries, dim ** -0.5))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shared", [576, 2560, 6400])
def test_every_merge(cuda, shared, dtype, dim):
    """Some three, a dozen and two dozen partials a head of 40 rows (one, two or all of a workgroup's threads a head)."""
    s = step(shared, [1 + i % 9 for i in range(40)], hq=16, hk=8, dim=dim, page=64, dtype=dtype, seed=shared)
    close(attend(cuda, shared, *s, dim ** -0.5), *want(*s, 1, dim ** -0.5))


@pytest.mark.parametrize("dim,page,rows", [(128, 16, 5), (64, 256, 5), (128, 48, 5), (128, 64, 70)])
def test_rows_that_do_not_see_the_prefix(cuda, dim, page, rows):
    """Padding rows get zeros; a row shorter than the shared keys is attended by itself through its own table, whatever
    its pages; one row's query that is no number stays in its row. Tables are wider than any row needs."""
    shared, hq, hk = 2 * 768 if page != 48 else 1440, 16, 4
    owns = [20] + [None, 40, 1, None, 7] * (rows // 5) + [33] * (rows - 1)
    q, k, v, tables, lens = step(shared, owns, hq=hq, hk=hk, dim=dim, page=page, dtype=torch.bfloat16, extra_width=5)
    lens[2] = shared // 2 + 3  # sees half the prefix
    lens[3] = shared - 1
    tables[3, :2] = tables[0, :2].flip(0)  # not the shared pages in the shared order
    q[len(owns) - 1] = math.nan
    scale = dim ** -0.5
    got = attend(cuda, shared, q, k, v, tables, lens, scale)
    y, a = want(q, k, v, tables, lens, 1, scale)
    close(got, y, a, slice(0, len(owns) - 1))
    assert got[-1].isnan().all()
    for i, n in enumerate(owns):
        if n is None:
            assert not got[i].any()


def test_only_padding_rows(cuda):
    """A captured graph's warmup: every table entry -1, every length 0."""
    for rows in (2, 100):
        k = torch.randn(4, 16, 2, 128, device=cuda).to(torch.bfloat16)
        q = torch.randn(rows, 8, 128, device=cuda).to(torch.bfloat16)
        ctx = Context(context_lens=torch.zeros(rows, dtype=torch.int32, device=cuda),
                      block_tables=torch.full((rows, 40), -1, dtype=torch.int32, device=cuda))
        assert not MI355XAttention(8, 128, 0.1, 2).decode_shared(q, k, k, ctx, 512).any()


def test_scores_that_rise_along_the_prefix(cuda):
    """Keys late in the prefix score hundreds of log2 units above the first ones, and some rows' own keys above those."""
    shared, owns, dim = 2048, [30, 60, 1, 200] * 12, 128
    q, k, v, tables, lens = step(shared, owns, hq=16, hk=4, dim=dim, page=64, dtype=torch.bfloat16)
    k[tables[0, 20].long()] *= 60
    k[tables[0, 31].long()] *= 90
    k[tables[5, 32].long(), :60] *= 120
    scale = dim ** -0.5
    sums = q.double().abs().amax((0, 1)) @ k.nan_to_num().double().abs().amax((0, 1, 2))
    close(attend(cuda, shared, q, k, v, tables, lens, scale), *want(q, k, v, tables, lens, 1, scale),
          score=min(0.1, 2 * dim * 2.0 ** -24 * sums.item() * scale))


def test_infinite_and_nan_keys(cuda):
    """A value that is not finite in the prefix reaches its dim in every row of its head, one in a row's own keys only that
    row, and what lies behind a row's keys in its last page none. (An infinite value comes out as infinity or as NaN: P V
    takes a probability as the sum of two 16-bit numbers, the second of either sign or zero, and inf - inf and 0 inf are
    NaN. The interface says so.)"""
    shared, owns, dim = 512, [20, 40, 9], 64
    q, k, v, tables, lens = step(shared, owns, hq=4, hk=2, dim=dim, page=16, dtype=torch.float16)
    v[tables[1, 32].long(), 3, 0, 5] = math.nan  # row 1's own key, kv head 0
    scale = dim ** -0.5
    got = attend(cuda, shared, q, k, v, tables, lens, scale)
    y, a = want(q, k, v, tables, lens, 1, scale)
    assert got[1, :2, 5].isnan().all() and got.isnan().sum() == 2
    fine = ~got.isnan().cpu()
    close(got.cpu()[fine], y[fine], a[fine])
    v[tables[0, 7].long(), 0, 1, 9] = math.inf  # the prefix, kv head 1
    got = attend(cuda, shared, q, k, v, tables, lens, scale)
    assert not got[:, 2:, 9].isfinite().any()
    got[:, 2:, 9], got[1, :2, 5] = 0, 0
    assert got.isfinite().all()


def test_strided_queries_and_outputs(cuda):
    shared, owns, hq, hk, dim = 1024, [50, 3, 77], 8, 4, 128
    s = step(shared, owns, hq=hq, hk=hk, dim=dim, page=32, dtype=torch.bfloat16)
    fused = torch.zeros(3, hq + 2 * hk, dim, dtype=torch.bfloat16, device=cuda)
    fused[:, :hq] = s[0].to(cuda)
    wide = torch.full((3, hq + 2, dim), 7.0, dtype=torch.bfloat16, device=cuda)
    scale = dim ** -0.5
    got = attend(cuda, shared, fused[:, :hq], *s[1:], scale, out=wide[:, 1:hq + 1])
    assert got.data_ptr() == wide[:, 1:].data_ptr() and (wide[:, [0, -1]] == 7).all()
    close(got, *want(*s, 1, scale))


def test_offsets_past_32_bits(cuda):
    """A pool of over 2^32 bytes a cache, the shared and own pages at its end."""
    hk, dim, page, blocks = 8, 128, 256, 9000  # 4.7 GB
    k, v = (torch.empty(blocks, page, hk, dim, dtype=torch.bfloat16, device=cuda) for _ in range(2))
    gen = torch.Generator(device=cuda).manual_seed(0)
    tail = 8980
    for c in (k, v):
        c[tail:] = torch.randn(blocks - tail, page, hk, dim, device=cuda, generator=gen).to(torch.bfloat16)
    tables = torch.tensor([[8999, 8990, 8981], [8999, 8990, 8985]], dtype=torch.int32)
    lens = torch.tensor([512 + 200, 512 + 3], dtype=torch.int32)
    q = torch.randn(2, 32, dim, device=cuda, generator=gen).to(torch.bfloat16)
    ctx = Context(context_lens=lens.to(cuda), block_tables=tables.to(cuda))
    got = MI355XAttention(32, dim, dim ** -0.5, hk).decode_shared(q, k, v, ctx, 512)
    close(got, *want(q.cpu(), k[tail:].cpu(), v[tail:].cpu(), tables - tail, lens, 1, dim ** -0.5))


def test_replays_in_graphs_and_on_streams(cuda):
    """Two captured graphs and eager calls on two streams at once: each call's partials are its own."""
    shared, dim, hq, hk, page = 2048, 128, 16, 8, 16
    backend, scale = MI355XAttention(hq, dim, dim ** -0.5, hk), dim ** -0.5
    steps, graphs = [], []
    for seed, owns in ((1, [40, 300, 1]), (2, [5] * 40)):
        q, k, v, tables, lens = step(shared, owns, hq=hq, hk=hk, dim=dim, page=page, dtype=torch.bfloat16, seed=seed)
        dev = [q.to(cuda), on(cuda, k), on(cuda, v), tables.to(cuda), lens.to(cuda)]
        y = want(q, k, v, tables, lens, 1, scale)
        ctx = Context(context_lens=dev[4], block_tables=dev[3])
        out = torch.empty_like(dev[0])
        backend.decode_shared(dev[0], dev[1], dev[2], ctx, shared, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            backend.decode_shared(dev[0], dev[1], dev[2], ctx, shared, out=out)
        steps.append((dev, ctx, out, y))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for turn in range(4):
        for dev, _, out, _ in steps:
            out.zero_()
        torch.cuda.synchronize()
        eager = []
        for stream, graph, (dev, ctx, _, _) in zip(streams, graphs, steps):
            with torch.cuda.stream(stream):
                graph.replay()
                eager.append(backend.decode_shared(dev[0], dev[1], dev[2], ctx, shared))
        torch.cuda.synchronize()
        for (dev, _, out, y), e in zip(steps, eager):
            close(out, *y)
            assert torch.equal(out, e)  # the same launches in the same order of sums
    steps[0][0][4].fill_(shared + 1)  # shorter rows, in the captured graph
    graphs[0].replay()
    q, k, v, tables, lens = (x.cpu() for x in steps[0][0])
    close(steps[0][2], *want(q, k, v, tables, lens, 1, scale))


def test_a_step_from_packing_to_attention(cuda):
    """The operators as a layer runs them: pack, rotate into the cache, attend the shared pages once; and the same step
    through store_kvcache and decode gives the same attention."""
    hq, hk, dim, page, prefix = 16, 4, 128, 16, 320
    gen = torch.Generator().manual_seed(3)
    shared_blocks = list(range(40, 40 + prefix // page))
    num_cached = [prefix + n for n in (0, 5, 16, 100, 31)]
    lists, at = [], 0
    for c in num_cached:
        own = -(-(c + 1 - prefix) // page)
        lists.append(shared_blocks + list(range(at, at + own)))
        at += own
    shared = shared_prefix_len(lists, num_cached, page)
    assert shared == prefix
    table = rotary_table(dim, 1024, device=cuda)
    k_cache, v_cache = (torch.randn(80, page, hk, dim, generator=gen).to(torch.bfloat16).to(cuda) for _ in range(2))
    other = k_cache.clone(), v_cache.clone()
    qkv = torch.randn(5, (hq + 2 * hk) * dim, generator=gen).to(torch.bfloat16).to(cuda)
    q, k, v = (x.view(5, -1, dim) for x in qkv.split([hq * dim, hk * dim, hk * dim], 1))
    positions, fields = Packer(cuda, page).pack(num_cached, [1] * 5, lists)
    assert fields.pop("order").tolist() == list(range(5))
    ctx = Context(**fields)
    backend = MI355XAttention(hq, dim, dim ** -0.5, hk)
    turned = backend.append_kvcache(q, k, v, k_cache, v_cache, ctx.slot_mapping, positions, table)
    got = backend.decode_shared(turned, k_cache, v_cache, ctx, shared)
    q2, k2 = apply_rotary(q, k, positions, table)
    backend.store_kvcache(k2, v.contiguous(), *other, ctx.slot_mapping)
    assert torch.equal(turned, q2) and torch.equal(k_cache, other[0]) and torch.equal(v_cache, other[1])
    y, a = want(turned.cpu(), k_cache.cpu(), v_cache.cpu(), ctx.block_tables.cpu(), ctx.context_lens.cpu(), 1, dim ** -0.5)
    close(got, y, a)
    close(backend.decode(q2, *other, ctx), y, a)
