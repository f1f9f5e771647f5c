"""Verification of drafted tokens against its 64-bit form: whole numbers, equal in every place."""
from __future__ import annotations

import importlib

import pytest

from conftest import PKG

torch = pytest.importorskip("torch")
import serving_refs as refs  # noqa: E402

pytestmark = pytest.mark.gpu
rt = importlib.import_module(f"{PKG}.runtime")


def inputs(batch, drafts, vocab, certain=False, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = 2.0 * torch.randn(batch, drafts + 1, vocab + pad, device="cuda", generator=g)
    target = torch.softmax(logits[..., :vocab], -1)
    draft = torch.softmax(logits[:, :drafts, :vocab] + torch.randn(batch, drafts, vocab, device="cuda", generator=g), -1)
    tokens = torch.zeros(batch, drafts, dtype=torch.int32, device="cuda")
    if drafts:
        tokens = torch.multinomial(draft.reshape(-1, vocab), 1, generator=g).reshape(batch, drafts).to(torch.int32)
    if pad:  # rows further apart than their length, poisoned between
        wide = torch.full((batch, drafts + 1, vocab + pad), float("nan"), device="cuda")
        wide[..., :vocab] = target
        target = wide[..., :vocab]
    u = torch.rand(batch, drafts + 1, device="cuda", generator=g)
    return target, None if certain else draft, tokens, u[:, :drafts].contiguous(), u[:, drafts].contiguous()


def run(ctx, target, draft, tokens, ua, us, counts=None):
    batch, rows, vocab = target.shape
    accepted = torch.full((batch,), 99, dtype=torch.int32, device="cuda")
    out = torch.full((batch, rows), 99, dtype=torch.int32, device="cuda")
    ctx.verify_drafts(target.data_ptr(), tokens.data_ptr(), ua.data_ptr(), us.data_ptr(), accepted.data_ptr(), out.data_ptr(),
                      batch, rows - 1, vocab, draft=0 if draft is None else draft.data_ptr(),
                      counts=0 if counts is None else counts.data_ptr(), ld_target=target.stride(1))
    ctx.sync()
    return accepted.cpu(), out.cpu()


def same(ctx, *args, counts=None):
    got = run(ctx, *args, counts=counts)
    want = refs.verify(args[0], args[1], args[2], None if counts is None else counts.cpu(), args[3], args[4])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    return got


@pytest.mark.parametrize("certain", [False, True])
@pytest.mark.parametrize("batch,drafts,vocab", [(1, 1, 1), (1, 0, 5), (3, 2, 2), (5, 4, 127), (2, 3, 129), (4, 5, 1000),
                                                (33, 7, 4097), (2, 40, 513), (3, 4, 50257), (70, 1, 300)])
def test_verify_matches(ctx, torch_cuda, certain, batch, drafts, vocab):
    for seed in range(3):
        same(ctx, *inputs(batch, drafts, vocab, certain, seed))


@pytest.mark.parametrize("batch,vocab", [(1, 65536), (1, 65537), (2, 70001), (18, 131071), (19, 100003)])
def test_verify_long_rows(ctx, torch_cuda, batch, vocab):
    """Around the row length and the number of sequences at which the blocks grow."""
    for certain in (False, True):
        same(ctx, *inputs(batch, 3, vocab, certain, seed=vocab))


def test_verify_counts_and_row_strides(ctx, torch_cuda):
    counts = torch.tensor([0, 1, 2, 3, 4, 9, -5], dtype=torch.int32, device="cuda")
    args = inputs(7, 4, 700, seed=3, pad=13)
    _, tokens = same(ctx, *args, counts=counts)
    assert (tokens[0, 1:] == -1).all()


def test_verify_all_taken_and_none(ctx, torch_cuda):
    target, _, tokens, ua, us = inputs(6, 3, 900, seed=5)
    accepted, _ = same(ctx, target, target[:, :3].contiguous(), tokens, ua, us)  # p = q: u q < p always
    assert (accepted == 3).all()
    tokens[:, 0] = torch.tensor([-1, 900, 2 ** 31 - 1, -(2 ** 31), -7, 901], device="cuda")  # outside the vocabulary
    accepted, _ = same(ctx, target, None, tokens, torch.zeros_like(ua), us)
    assert (accepted == 0).all()


def test_verify_nothing_left_draws_from_target(ctx, torch_cuda):
    """p below q everywhere but refused: the rest is empty and the draw is from p; an empty p gives -1."""
    target = torch.zeros(3, 2, 64, device="cuda")
    target[0, 0, 5:9] = 0.25
    target[1, 0, 63] = 2.0 ** -149  # the smallest number is a step too
    draft = torch.full((3, 1, 64), 0.5, device="cuda")
    args = (target, draft, torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.full((3, 1), 0.999, device="cuda"),
            torch.tensor([0.6, 0.9, 0.3], device="cuda"))
    accepted, tokens = same(ctx, *args)
    assert accepted.tolist() == [0, 0, 0] and tokens[:, 0].tolist() == [7, 63, -1]


def test_verify_edges_of_the_steps(ctx, torch_cuda):
    """Thresholds on a step's edge go to the next step; u = 0 takes the first that holds anything."""
    target = torch.zeros(5, 1, 4096, device="cuda")
    target[:, 0, 1024::1024] = 0.25
    target[:, 0, 7] = 0.25
    us = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], device="cuda")
    empty = torch.zeros(5, 0, device="cuda")
    _, tokens = same(ctx, target, None, empty.to(torch.int32), empty, us)
    assert tokens[:, 0].tolist() == [7, 1024, 2048, 3 * 1024, 3 * 1024]


def test_verify_follows_the_target(ctx, torch_cuda):
    """Over many draws of drafts and numbers the emitted first token is distributed as the target says."""
    torch.manual_seed(0)
    n, vocab = 60000, 6
    p, q = torch.tensor([.3, .05, .25, .1, .2, .1]), torch.tensor([.1, .4, .1, .2, .1, .1])
    target, draft = p.cuda().expand(n, 2, vocab).contiguous(), q.cuda().expand(n, 1, vocab).contiguous()
    drafted = torch.multinomial(q.cuda(), n, replacement=True).to(torch.int32)[:, None].contiguous()
    _, tokens = run(ctx, target, draft, drafted, torch.rand(n, 1, device="cuda"), torch.rand(n, device="cuda"))
    share = torch.bincount(tokens[:, 0].long(), minlength=vocab).double() / n
    assert ((share - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / n).sqrt()).all()  # five deviations


def test_verify_refusals(ctx, torch_cuda):
    x = torch.zeros(64, device="cuda")
    i = torch.zeros(64, dtype=torch.int32, device="cuda")
    good = dict(target=x.data_ptr(), drafted=i.data_ptr(), u_accept=x.data_ptr(), u_sample=x.data_ptr(),
                accepted=i.data_ptr() + 64, tokens=i.data_ptr() + 128, batch=1, drafts=1, vocab=4)
    for kw in (dict(target=0), dict(drafted=0), dict(u_accept=0), dict(u_sample=0), dict(accepted=0), dict(tokens=0),
               dict(batch=-1), dict(drafts=-1), dict(vocab=0), dict(ld_target=3), dict(draft=x.data_ptr(), ld_draft=3),
               dict(batch=2 ** 31), dict(vocab=2 ** 31 - 1, ld_target=2 ** 31), dict(target=x.data_ptr() + 2), dict(tokens=i.data_ptr() + 1),
               dict(tokens=i.data_ptr()), dict(tokens=i.data_ptr() + 64),
               dict(counts=i.data_ptr() + 2)):
        with pytest.raises(rt.B2KError) as e:
            ctx.verify_drafts(**{**good, **kw})
        assert e.value.status == rt.B2K_EINVAL
    ctx.verify_drafts(**{**good, "batch": 0, "target": 0})
    ctx.sync()
