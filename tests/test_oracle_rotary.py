"""The rotary oracle and the frequencies on the CPU: closed forms, properties of a rotation, known values, refusals."""

import math

import pytest
import torch

import lvattn
from oracle import rotary as R

SCALINGS = [None, dict(rope_type="linear", factor=4.0), dict(rope_type="ntk", factor=8.0),
            dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192),
            dict(rope_type="llama3", factor=32.0, low_freq_factor=1.0, high_freq_factor=4.0,
                 original_max_position_embeddings=8192),
            dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768),
            dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096, beta_fast=32, beta_slow=1,
                 attention_factor=1.0),
            dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096, mscale=1.0, mscale_all_dim=0.707),
            dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096, truncate=False)]


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_score_depends_on_the_distance_alone(interleaved):
    gen = torch.Generator().manual_seed(0)
    q, k = (torch.randn(1, 1, 16, generator=gen).double() for _ in range(2))

    def score(m, n):
        a, _ = R.rotate(q, torch.tensor([m]), 16, interleaved=interleaved)
        b, _ = R.rotate(k, torch.tensor([n]), 16, interleaved=interleaved)
        return (a * b).sum().item()

    assert score(5, 2) == pytest.approx(score(105, 102), abs=1e-9)
    assert abs(score(5, 2) - score(5, 3)) > 1e-3
    assert score(0, 0) == pytest.approx((q * k).sum().item())


def test_closed_forms():
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]]])
    y, _ = R.rotate(x, torch.tensor([0]), 4)
    assert torch.equal(y, x.double())  # position 0 turns nothing
    y, _ = R.rotate(x, torch.tensor([3]), 2)  # one pair, angle 3: dims 0 and 1 in either layout
    c, s = math.cos(3), math.sin(3)
    assert y.flatten().tolist() == pytest.approx([c - 2 * s, 2 * c + s, 3, 4, 5, 6])
    half, _ = R.rotate(x, torch.tensor([7]), 4)
    inter, _ = R.rotate(x[..., [0, 2, 1, 3, 4, 5]], torch.tensor([7]), 4, interleaved=True)
    assert torch.allclose(half, inter[..., [0, 2, 1, 3, 4, 5]])  # the layouts differ in the order of dims only
    y, _ = R.rotate(x, torch.tensor([0]), 2, weight=torch.full((6,), 2.0), eps=0.0)
    assert y.pow(2).mean().item() == pytest.approx(4.0)


@pytest.mark.parametrize("scaling", SCALINGS)
@pytest.mark.parametrize("rotary_dim,base", [(128, 1e6), (64, 1e4), (20, 5e5)])
def test_frequencies_match_the_oracle(scaling, rotary_dim, base):
    want, amp = R.angles(rotary_dim, base, scaling)
    got, got_amp = lvattn.rotary_frequencies(rotary_dim, base, scaling)
    assert got.dtype.name == "float64" and got.tolist() == pytest.approx(want, rel=1e-12) and got_amp == amp
    table = lvattn.rotary_table(rotary_dim, 70_000, base, scaling, device="cpu")
    assert table.shape == (70_000, rotary_dim) and table.dtype == torch.float32
    for pos in (0, 1, 65_535, 65_536, 69_999):
        exact = [amp * math.cos(pos * w) for w in want] + [amp * math.sin(pos * w) for w in want]
        assert (table[pos].double() - torch.tensor(exact, dtype=torch.float64)).abs().max() <= 2.0 ** -24 * max(amp, 1) * 1.5


def test_the_ends_of_the_scalings():
    plain, _ = lvattn.rotary_frequencies(128, 5e5)
    for s in SCALINGS[3:]:
        scaled, _ = lvattn.rotary_frequencies(128, 5e5, s)
        assert scaled[0] == plain[0] and scaled[-1] == pytest.approx(plain[-1] / s["factor"])
    ntk, _ = lvattn.rotary_frequencies(128, 5e5, SCALINGS[2])
    assert ntk[0] == 1.0 and ntk[-1] == pytest.approx(plain[-1] / 8.0)


@pytest.mark.parametrize("args,message", [
    ((7,), "not a positive even"), ((0,), "not a positive even"), ((8, 1.0), "not above 1"),
    ((8, 1e4, dict(rope_type="spline", factor=2.0)), "rope_type 'spline'"),
    ((8, 1e4, dict(rope_type="linear", factor=2.0, mscale=1.0)), "takes no mscale"), ((8, 1e4, dict(factor=2.0)), "takes no"),
    ((8, 1e4, dict(rope_type="linear")), "factor of at least 1"),
    ((8, 1e4, dict(rope_type="linear", factor=0.5)), "factor of at least 1"),
    ((2, 1e4, dict(rope_type="ntk", factor=2.0)), "width above 2"),
    ((8, 1e4, dict(rope_type="yarn", factor=2.0)), "original_max_position_embeddings"),
    ((8, 1e4, dict(rope_type="yarn", factor=2.0, original_max_position_embeddings=64, beta_fast=1, beta_slow=2)), "beta"),
    ((8, 1e4, dict(rope_type="llama3", factor=2.0, original_max_position_embeddings=64, low_freq_factor=4)), "low_freq"),
])
def test_frequencies_refuse(args, message):
    with pytest.raises(ValueError, match=message):
        lvattn.rotary_frequencies(*args)
    with pytest.raises(ValueError, match="0 positions"):
        lvattn.rotary_table(8, 0, device="cpu")


def heads(t=4, h=2, d=16, dtype=torch.bfloat16):
    return torch.zeros(t, h, d, dtype=dtype)


POS, TABLE = torch.zeros(4, dtype=torch.int64), torch.zeros(32, 16)


@pytest.mark.parametrize("q,k,positions,table,message", [
    (None, None, POS, TABLE, "no heads"),
    (heads(dtype=torch.float32), None, POS, TABLE, "bf16 or fp16"),
    (heads()[0], None, POS, TABLE, "bf16 or fp16"),
    (heads(), heads(t=3), POS, TABLE, "k is"),
    (heads(), heads(d=32), POS, TABLE, "k is"),
    (heads(), heads(dtype=torch.float16), POS, TABLE, "k is"),
    (heads().transpose(1, 2), None, POS, TABLE, "unit dim stride"),
    (heads(), heads(), POS.int(), TABLE, "positions must be"),
    (heads(), heads(), POS[:3], TABLE, "positions must be"),
    (heads(), heads(), torch.zeros(8, dtype=torch.int64)[::2], TABLE, "positions must be"),
    (heads(), heads(), POS, TABLE.double(), "the table must be"),
    (heads(), heads(), POS, torch.zeros(32, 18), "the table must be"),
    (heads(), heads(), POS, torch.zeros(32, 7), "the table must be"),
    (heads(), heads(), POS, TABLE.t().contiguous().t(), "the table must be"),
    (heads(), heads(), POS, TABLE[:0], "the table must be"),
    (heads(), heads(), POS, TABLE, "must be on one GPU"),
])
def test_calls_refuse(q, k, positions, table, message):
    with pytest.raises(ValueError, match=message):
        lvattn.apply_rotary(q, k, positions, table)


def test_outputs_refuse():
    for out, message in ((heads(t=3), "out_q is"), (heads(dtype=torch.float16), "must be on one GPU|out_q is"),
                         (heads(t=1).expand(4, 2, 16), "holds one row")):
        q = heads()
        with pytest.raises(ValueError, match=message):
            lvattn.rotary.output_heads("apply_rotary", "out_q", q, out, (4, 16, torch.bfloat16, -1))
    with pytest.raises(ValueError, match="its input missing"):
        lvattn.rotary.output_heads("apply_rotary", "out_k", None, heads(), (4, 16, torch.bfloat16, -1))


def test_norms_and_appends_refuse():
    w = torch.ones(16, dtype=torch.bfloat16)
    for bad in (w.float(), w[:8], torch.ones(32, dtype=torch.bfloat16)[::2]):
        with pytest.raises(ValueError, match="q_weight must be"):
            lvattn.norm_rotary(heads(), heads(), bad, w, POS, TABLE)
    backend = lvattn.MI355XAttention(4, 16, 1.0, 2)
    cache = torch.zeros(3, 16, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k is|v is"):
        backend.append_kvcache(None, heads(), heads(t=3), cache, cache, POS.int(), POS, TABLE)
    with pytest.raises(ValueError, match="must be on one GPU"):
        backend.append_kvcache(heads(), heads(), heads(), cache, cache, POS.int(), POS, TABLE)


def test_the_c_entries_refuse():
    from lvattn import _capi

    def rotary(*, rot=16, dim=16, hq=2, hkv=2, tokens=4, positions=64, eps=0.0, dtype=0, q=16, weight=None):
        _capi.call("lv_rotary", q, 32, 16, 16, 32, 16, 16, 16, positions, rot, 0, weight, None, eps, tokens, hq, hkv,
                   dim, 16, 32, 16, 16, 32, 16, dtype, None)

    for args, message in [(dict(rot=7), "rotary width 7 must be even"), (dict(rot=18), "at most the head width 16"),
                          (dict(dtype=2), "not bf16 or fp16"), (dict(hq=0, hkv=0), "bad sizes"),
                          (dict(tokens=-1), "bad sizes"), (dict(positions=0), "a table of 0 positions"),
                          (dict(q=None), "null pointer"), (dict(eps=-1.0, weight=16), "eps must not be negative"),
                          (dict(tokens=(1 << 31) - 1, hq=64), "larger than one launch")]:
        with pytest.raises(_capi.LvError, match=message):
            rotary(**args)
    rotary(tokens=0)

    def append(*, block=16, hkv=2, slots=16, tokens=4):
        _capi.call("lv_append_kvcache", 16, 32, 16, 16, 32, 16, 16, 32, 16, 16, 16, 64, 16, 0, None, None, 0.0, tokens,
                   2, hkv, 16, 16, 32, 16, 16, 16, 512, 32, 16, block, slots, 0, None)

    for args, message in [(dict(block=0), "block_size must be positive"), (dict(hkv=0), "no key heads"),
                          (dict(slots=None), "null pointer")]:
        with pytest.raises(_capi.LvError, match=message):
            append(**args)
    append(tokens=0)
