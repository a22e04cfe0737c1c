"""``verify_draft`` on rows that are read and hold a NaN: a NaN counts as -inf."""

import math

import pytest
import torch

import logits_plain as plain
from lattice_based_tagger_amd import logits

pytestmark = pytest.mark.gpu

INF = math.inf


def check(a):
    """The tokens and accepted counts of the same call with -inf for every NaN,
    which the plain form in 64 bits gives too; whole numbers, so equal."""
    clean = {k: torch.where(v.isnan(), -INF, v) if k in ('target', 'draft') and v is not None else v
             for k, v in a.items()}
    tokens, accepted = plain.verify(clean['target'], clean['draft_ids'], clean['accept_u'], clean['sample_u'],
                                    clean['draft'])
    got, same = logits.verify_draft(**a), logits.verify_draft(**clean)
    assert torch.equal(same.accepted.cpu(), accepted) and torch.equal(same.tokens.cpu(), tokens)
    assert torch.equal(got.accepted.cpu(), accepted) and torch.equal(got.tokens.cpu(), tokens)
    return got


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('certain', [False, True])
@pytest.mark.parametrize('batch, drafts, vocab', [(24, 3, 41), (24, 3, 1000), (24, 2, 40001), (3, 2, 300007)])
def test_nan_in_a_row_that_counts(dtype, certain, batch, drafts, vocab):
    """One NaN, or many, anywhere in a target's row, a drafter's or both: beside
    the drafted token, first, last, and at the drafted token itself."""
    g = torch.Generator().manual_seed(vocab + batch)
    target = (torch.randn(batch, drafts + 1, vocab, generator=g) * 2).to(dtype).cuda()
    best = target.float().argmax(-1)
    target.scatter_add_(2, best[..., None], torch.full_like(best[..., None], 6, dtype=dtype))
    ids = best[:, :drafts].clone()
    draft = None if certain else (target[:, :drafts].float() +
                                  0.5 * torch.randn(batch, drafts, vocab, generator=g).cuda()).to(dtype)
    place = torch.arange(vocab, device='cuda')
    other = (ids + 1 + torch.arange(drafts, device='cuda')) % vocab
    for b in range(batch):
        kind = b % 8
        rows = [target] if kind < 3 or certain else [draft] if kind < 6 else [target, draft]
        for x in rows:
            for i in range(drafts):
                if kind % 3 == 0:
                    x[b, i, other[b, i]] = math.nan
                elif kind % 3 == 1:
                    x[b, i, 0] = math.nan
                    x[b, i, -1] = math.nan
                else:
                    x[b, i, (place % 3 == 1) & (place != ids[b, i])] = math.nan
    target[0, 0, ids[0, 0]] = math.nan                  # never accepted
    target[1, drafts, 2::5] = math.nan                  # the place behind the last draft
    if not certain:
        draft[2, 0, ids[2, 0]] = math.nan               # q = 0
    a = dict(target=target, draft_ids=ids, accept_u=torch.rand(batch, drafts, generator=g).cuda(),
             sample_u=torch.rand(batch, generator=g).cuda(), draft=draft)
    got = check(a)
    assert got.accepted[0] == 0 and (batch < 8 or got.accepted.max() == drafts)
    # accepted and refused by numbers beside their ends: the row's NaN decides nothing
    a['accept_u'] = torch.full_like(a['accept_u'], 1 - 2.0 ** -24)
    check(a)
    a['accept_u'] = torch.full_like(a['accept_u'], 2.0 ** -20)
    check(a)


@pytest.mark.parametrize('certain, batch, drafts, vocab', [(False, 300, 7, 131072), (True, 180, 8, 200003)])
def test_nan_place_by_place(certain, batch, drafts, vocab):
    """The same in batches so large that they are taken a place at a time."""
    dtype = torch.float32 if certain else torch.bfloat16
    g = torch.Generator('cuda').manual_seed(batch)
    x = torch.empty(batch, drafts + 1, vocab, dtype=dtype, device='cuda').normal_(0, 2, generator=g)
    best = x.argmax(-1, keepdim=True)
    x.scatter_add_(2, best, torch.full_like(best, 9, dtype=dtype))
    ids = best[:, :drafts, 0].clone()
    draft = None if certain else x[:, :drafts].clone()
    if draft is not None:
        draft[3::4] += torch.empty_like(draft[3::4]).normal_(0, 0.3, generator=g)
    off = (ids + 7) % vocab
    x[::3, :drafts].scatter_(2, off[::3, :, None], math.nan)
    x[1::9, drafts, 5] = math.nan
    if draft is not None:
        draft[1::3].scatter_(2, off[1::3, :, None], math.nan)
    u = torch.rand(batch, drafts, generator=g, device='cuda')
    clean = [None if t is None else torch.where(t.isnan(), -INF, t) for t in (x, draft)]
    rest = dict(draft_ids=ids, accept_u=u, sample_u=torch.rand(batch, generator=g, device='cuda'))
    got = logits.verify_draft(target=x, draft=draft, **rest)
    same = logits.verify_draft(target=clean[0], draft=clean[1], **rest)
    assert torch.equal(got.accepted, same.accepted) and torch.equal(got.tokens, same.tokens)
    cut = lambda t, n=24: None if t is None else t[:n]
    tokens, accepted = plain.verify(cut(clean[0]), cut(ids), cut(u), cut(rest['sample_u']), cut(clean[1]))
    assert torch.equal(got.accepted[:24].cpu(), accepted) and torch.equal(got.tokens[:24].cpu(), tokens)
    assert got.accepted.max() == drafts and got.accepted.min() < drafts


@pytest.mark.parametrize('certain', [False, True])
def test_a_row_of_nan(certain):
    """Nothing but NaN: as a row of -inf, from which no token is drawn."""
    target = torch.randn(4, 2, 300, generator=torch.Generator().manual_seed(1)).cuda()
    draft = None if certain else target[:, :1].clone()
    target[0, 0] = math.nan
    target[1, 1] = math.nan
    if draft is not None:
        draft[2] = math.nan
    ids = target[:, :1].nan_to_num().argmax(-1)
    got = check(dict(target=target, draft_ids=ids, accept_u=torch.full((4, 1), 0.001).cuda(),
                     sample_u=torch.rand(4, generator=torch.Generator().manual_seed(2)).cuda(), draft=draft))
    assert got.tokens[0].tolist() == [-1, -1] and got.tokens[1, 1] == -1


@pytest.mark.parametrize('certain', [False, True])
@pytest.mark.parametrize('vocab, seed', [(9000, 1), (40000, 2), (131072, 3)])
def test_close_to_the_line(certain, vocab, seed):
    """Random numbers within a few steps of 32 bits of p / q on either side, of rows
    whose every thread begins 2^31 below its largest: decided as by 64 bits."""
    g = torch.Generator().manual_seed(seed)
    batch, temperature = 64, 0.7317
    def rows():
        x = torch.rand(batch, 2, vocab, generator=g) * 0.3
        # a block's first steps of every chunk it may begin at
        x[:, :, (torch.arange(vocab) // 4096) % 2 == 0] -= 31 * math.log(2) * temperature
        return x
    target = rows()
    ids = torch.randint(4096, 8192, (batch, 1), generator=g)
    target[torch.arange(batch), 0, ids[:, 0]] += 11.0
    draft = None
    p = torch.softmax(target[:, 0].double() / temperature, -1).gather(1, ids)[:, 0]
    q = torch.ones_like(p)
    if not certain:
        draft = rows()[:, :1]
        draft[torch.arange(batch), 0, ids[:, 0]] += 11.5
        q = torch.softmax(draft[:, 0].double() / temperature, -1).gather(1, ids)[:, 0]
    u = (p / q).clamp(max=1 - 2.0 ** -23).float()
    for step in range(-3, 4):
        near = u.clone()
        for _ in range(abs(step)):
            near = torch.nextafter(near, torch.tensor(2.0 if step > 0 else -1.0)).clamp(max=1 - 2.0 ** -24)
        a = dict(target=target.cuda(), draft_ids=ids.cuda(), accept_u=near[:, None].cuda(),
                 sample_u=torch.rand(batch, generator=g).cuda(), draft=None if certain else draft.cuda())
        got = logits.verify_draft(temperature=temperature, **a)
        # (64-bit sums decide: p of the plain form is within 1e-12 of the kernel's)
        clear = (near.double() * q - p).abs() > 1e-10 * p
        assert torch.equal(got.accepted.cpu()[clear], (near.double() * q < p)[clear].long())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('certain', [False, True])
@pytest.mark.parametrize('drafts', [255, 256])
def test_the_most_drafts(dtype, certain, drafts):
    """As many as a call takes, a place more than a block has threads: none, some and
    all of them accepted, with and without lengths."""
    g = torch.Generator().manual_seed(drafts)
    batch, vocab = 6, 70
    target = torch.randn(batch, drafts + 1, vocab, generator=g).to(dtype).cuda()
    ids = target[:, :drafts].float().argmax(-1)
    target.scatter_add_(2, ids[..., None], torch.full(ids[..., None].shape, 12, dtype=dtype, device='cuda'))
    draft = None if certain else target[:, :drafts].clone()
    u = torch.full((batch, drafts), 0.5)
    if not certain:
        draft[1, drafts - 1, ids[1, drafts - 1]] += 30     # (surer than the target: still accepted, p is near 1)
    ids[2, 0] = vocab                                      # none
    ids[3, drafts - 1] = vocab                             # all but the last
    ids[4, drafts // 2] = -1
    a = dict(target=target, draft_ids=ids, accept_u=u.cuda(), sample_u=torch.rand(batch, generator=g).cuda(), draft=draft)
    got = check(a)
    assert got.accepted.tolist() == [drafts, drafts, 0, drafts - 1, drafts // 2, drafts]
    n = torch.tensor([drafts, drafts - 1, 5, drafts, 0, 200], dtype=torch.int32)
    tokens, accepted = plain.verify(target, ids, u, a['sample_u'], draft, n)
    got = logits.verify_draft(lengths=n.cuda(), **a)
    assert torch.equal(got.accepted.cpu(), accepted) and torch.equal(got.tokens.cpu(), tokens)


def test_lengths_beyond_their_ends():
    """Lengths are taken as within [0, drafts]."""
    g = torch.Generator().manual_seed(9)
    target = torch.randn(5, 4, 100, generator=g).cuda()
    ids = target[:, :3].argmax(-1)
    target.scatter_add_(2, ids[..., None], torch.full((5, 3, 1), 9.0, device='cuda'))
    u, s = torch.full((5, 3), 0.01).cuda(), torch.rand(5, generator=g).cuda()
    n = torch.tensor([-1, -2 ** 31, 4, 2 ** 31 - 1, 2], dtype=torch.int32)
    got = logits.verify_draft(target, ids, u, s, lengths=n.cuda())
    tokens, accepted = plain.verify(target, ids, u, s, None, n.clamp(0, 3))
    assert torch.equal(got.accepted.cpu(), accepted) and torch.equal(got.tokens.cpu(), tokens)
    assert got.accepted.tolist() == [0, 0, 3, 3, 2]
