"""Logits that are signalling NaN, as memory may hold them: they count as any NaN."""

import math

import pytest
import torch

import logits_plain as plain
from lattice_based_tagger_amd import logits

pytestmark = pytest.mark.gpu

INF = math.inf
TYPES = [torch.float32, torch.float16, torch.bfloat16]
BITS = {torch.float32: (torch.int32, 0x7f800001), torch.float16: (torch.int16, 0x7c01), torch.bfloat16: (torch.int16, 0x7f81)}


def put(x, at):
    """x with a signalling NaN where ``at`` is true (as bits: arithmetic would quiet it)."""
    whole, bits = BITS[x.dtype]
    return torch.where(at, torch.tensor(bits, dtype=whole, device=x.device), x.view(whole)).view(x.dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, k', [
    (16500, 41, 5), (8, 41, 9), (8, 100, 3), (8, 200, 40), (8, 700, 100), (8, 2000, 64), (8, 4000, 256), (2100, 8000, 20),
    (600, 20000, 100), (8, 40000, 256), (8, 140000, 20)])
def test_top(dtype, rows, vocab, k):
    """Beside the best logits and everywhere, one in a row, and beside an infinity."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).cuda()
    best = x.topk(min(k, vocab // 8)).indices
    at = torch.zeros(rows, vocab, dtype=torch.bool, device='cuda')
    for off in (1, 2, 3):
        at[off::8].scatter_(1, (best[off::8] + off) % vocab, True)
    at[4::8] = torch.rand(vocab, generator=g).cuda() < 0.7
    at[5::8, vocab // 2] = True
    at[6] = True
    x[7, 3] = INF
    at[7, 2] = at[7, 4] = True
    x = put(x, at)
    assert (x.isnan() == at).all()
    got = logits.top_logits(x, k)
    values, ids, lse = plain.top_logits(x, k)
    assert torch.equal(got.ids.cpu(), ids)
    same = (got.values.double().cpu() == values) | (got.values.isnan().cpu() & values.isnan())
    assert same.all()
    lse_at = got.lse.double().cpu()
    tol = plain.lse_tolerance(torch.where(lse.isfinite(), lse, 0.0), vocab)
    assert (((lse_at - lse).abs() <= tol) | (lse_at == lse) | (lse_at.isnan() & lse.isnan())).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('certain', [False, True])
def test_verify(dtype, certain):
    """As -inf, whatever lies beside it: at a temperature where a logit next to the
    largest is far below it."""
    g = torch.Generator().manual_seed(6)
    batch, drafts, vocab = 16, 3, 5000
    target = (torch.randn(batch, drafts + 1, vocab, generator=g) * 3).to(dtype).cuda()
    best = target.float().argmax(-1, keepdim=True)
    target.scatter_add_(2, best, torch.full_like(best, 60, dtype=dtype))
    ids = best[:, :drafts, 0].contiguous()
    draft = None if certain else target[:, :drafts].clone()
    at = torch.zeros(batch, drafts + 1, vocab, dtype=torch.bool, device='cuda')
    at[:, :, ::3].scatter_(2, (best // 3 + 1) % (vocab // 3), True)
    at.scatter_(2, (best + 1) % vocab, True)
    at.scatter_(2, best, False)
    args = dict(draft_ids=ids, accept_u=torch.rand(batch, drafts, generator=g).cuda(),
                sample_u=torch.rand(batch, generator=g).cuda(), temperature=0.5)
    clean = torch.where(at, -INF, target)
    low = None if certain else torch.where(at[:, :drafts], -INF, draft)
    tokens, accepted = plain.verify(clean, ids, args['accept_u'], args['sample_u'], low, None, 0.5)
    got = logits.verify_draft(target=put(target, at), draft=None if certain else put(draft, at[:, :drafts]), **args)
    assert torch.equal(got.accepted.cpu(), accepted) and torch.equal(got.tokens.cpu(), tokens)
