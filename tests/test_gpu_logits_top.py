"""``top_logits`` where a bound that a row's logits are cut at falls on zero, and
the sign of zeros."""

import pytest
import torch

import logits_plain as plain
from lattice_based_tagger_amd import logits

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def check(x, k):
    got = logits.top_logits(x, k)
    values, ids, _ = plain.top_logits(x, k)
    assert torch.equal(got.ids.cpu(), ids)
    assert torch.equal(got.values.double().cpu(), values)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, k, threads', [
    (2100, 8192, 32, 64), (600, 20000, 100, 256), (3, 40000, 100, 512), (600, 40000, 200, 512), (2, 140000, 100, 512)])
def test_a_cut_at_zero(dtype, rows, vocab, k, threads):
    """Of a step that rises above all before it, zeros come as the k best of what
    is cut first -- every thread's second logit --, then zeros of lower indices, in
    the threads' later ones."""
    e = 16 // dtype.itemsize
    step = threads * 4 * e
    row = torch.full((vocab,), -1.0)
    row[:step] = -2.0
    row[step] = -1.5
    place = torch.arange(vocab)
    j, at = (place - step) // e, (place - step) % e
    some = min(k, threads // 2)
    row[(place >= step) & (at == 1) & (j >= some // 2) & (j < some // 2 + k)] = 0.0
    row[(place >= step) & (at == e - 1) & (j < some // 2)] = 0.0
    x = row.to(dtype).cuda().expand(rows, vocab).contiguous()
    x[1] += 1
    x[-1] = -x[-1]
    check(x, k)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, k', [(2100, 8000, 30), (600, 20000, 100), (40, 40000, 256), (3, 200000, 60)])
def test_rising_ties_about_zero(dtype, rows, vocab, k):
    """A few values, rarer the larger they are and rising along the row, 0 the
    largest or in their middle."""
    g = torch.Generator().manual_seed(vocab)
    x = -torch.rand(rows, vocab, generator=g).pow(3).mul(4).floor()
    x -= torch.arange(vocab).mul(-4.0 / vocab).add(4).floor() * (torch.rand(rows, 1, generator=g) < 0.7)
    x[torch.rand(rows, vocab, generator=g) < 2.0 * k / vocab] = 0.0
    x[::3] += 1
    check(x.to(dtype).cuda(), k)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, k', [
    (16500, 41, 1), (16500, 41, 5), (16500, 60, 8), (7, 41, 9), (7, 100, 3), (7, 200, 40), (7, 700, 100), (7, 2000, 64),
    (2100, 7000, 20), (600, 9000, 100), (5, 9000, 256), (5, 40000, 256), (3, 140000, 20)])
def test_the_sign_of_zeros(dtype, rows, vocab, k):
    """-0 and 0 are equal, by their indices; each comes back as it is."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randint(-3, 1, (rows, vocab), generator=g).float()
    x = torch.where(torch.rand(rows, vocab, generator=g) < 0.5, x.abs().neg(), x)
    x[0] = -0.0
    x[1, ::2] = -x[1, ::2].abs()
    x[2, 3:] = -0.0
    assert (x == 0).any() and x[0].signbit().all()
    x = x.to(dtype).cuda()
    check(x, k)
    got = logits.top_logits(x, k)
    assert torch.equal(got.values.float().signbit(), x.gather(1, got.ids).float().signbit())
    assert got.values[0].float().signbit().all()
