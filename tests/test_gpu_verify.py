"""The check of drafted tokens on the GPU, against its definition in 64 bits."""

import pytest
import torch

import b200_attention as b2
from b200_attention import check_device_errors, clear_device_errors, read_device_errors
from cache4_reference import verify64

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.fixture(autouse=True)
def no_reports_left():
    yield
    clear_device_errors(DEV)


def parents_of(B, T, shape, gen):
    if shape == "chain":
        return None
    if shape == "star":  # all nodes are the root's children
        return torch.zeros(T, dtype=torch.int32)
    p = torch.full((B, T), -1, dtype=torch.int32)
    for i in range(1, T):
        p[:, i] = torch.randint(max(0, i - 4), i, (B,), generator=gen, dtype=torch.int32)
    return p


def case(B, T, V, shape, drafter, dtype=torch.float32, ragged=False, seed=0, spread=4.0):
    gen = torch.Generator().manual_seed(seed * 100 + V + T)
    logits = spread * torch.randn(B, T, V, generator=gen)
    near = torch.softmax(logits[:, :max(1, T - 1)] + torch.randn(B, max(1, T - 1), V, generator=gen), -1)
    parents = parents_of(B, T, shape, gen)
    at = (torch.arange(T) - 1).expand(B, T) if parents is None else parents.expand(B, T)
    tokens = torch.randint(0, V, (B, T), generator=gen)
    for b in range(B):
        for i in range(1, T):
            tokens[b, i] = torch.multinomial(near[b, at[b, i]], 1, generator=gen)
    drafts = torch.tensor([max(0, T - 2 * b) for b in range(B)], dtype=torch.int32) if ragged else None
    return dict(logits=logits.to(dtype), tokens=tokens, uniforms=torch.rand(B, T, generator=gen),
                draft_probs=near[:, :T - 1] if drafter else None, parents=parents, draft_lens=drafts)


def run(c, **kw):
    on = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in c.items()}
    out = b2.b200_verify_drafts(**on, **kw)
    check_device_errors(DEV)
    return out


def check(c, temperature=1.0):
    paths, counts, following = run(c, temperature=temperature)
    want = verify64(c["logits"], c["tokens"], c["uniforms"], c["draft_probs"], c["parents"],
                    c["draft_lens"], temperature)
    assert paths.dtype == torch.int32 and counts.dtype == torch.int32 and following.dtype == torch.int64
    assert torch.equal(counts.cpu(), want[1])
    assert torch.equal(paths.cpu(), want[0])
    assert torch.equal(following.cpu(), want[2])
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("B,T,V,shape,ragged", [
    (1, 1, 1, "chain", False),
    (2, 1, 7, "chain", False),
    (5, 4, 50, "chain", True),
    (7, 12, 333, "tree", False),
    (9, 9, 16, "star", True),
    (4, 6, 5001, "tree", True),
    (3, 5, 20001, "tree", False),
    (6, 8, 32000, "chain", False),
])
def test_against_the_definition(B, T, V, shape, ragged, drafter, dtype):
    c = case(B, T, V, shape, drafter, dtype, ragged)
    for temperature in (1.0, 0.6, 0.0):
        check(c, temperature)


def test_many_draws_of_next_tokens():
    """A flat distribution: each draw sits next to many borders of the cumulated weights."""
    for seed in range(4):
        check(case(64, 2, 32000, "chain", seed % 2 == 0, seed=seed, spread=1.0), 1.0)
    check(case(40, 7, 100003, "tree", True, seed=9, spread=2.0), 0.9)


def test_refusals_of_siblings_and_of_the_same_token_twice():
    for seed in range(6):
        c = case(16, 17, 40, "star", True, seed=seed, spread=1.0)
        c["tokens"][:, 3] = c["tokens"][:, 2]
        c["tokens"][:, 9] = c["tokens"][:, 1]
        c["uniforms"][:, 1:] = c["uniforms"][:, 1:] * 0.2 + 0.8
        check(c)
        check(dict(c, draft_probs=None))


def test_tokens_are_distributed_as_the_targets():
    """The next token after the root, over many random numbers: within 5 standard deviations of the
    target's probability, with drafts that are unlike the target."""
    gen = torch.Generator().manual_seed(1)
    B, T, V = 60000, 4, 6
    logits = torch.randn(1, T, V, generator=gen).expand(B, T, V)
    near = torch.softmax(torch.randn(1, T - 1, V, generator=gen), -1).expand(B, T - 1, V)
    parents = torch.zeros(T, dtype=torch.int32)
    tokens = torch.zeros(B, T, dtype=torch.int64)
    tokens[:, 1:] = torch.multinomial(near[0, 0], B * 3, replacement=True, generator=gen).view(B, 3)
    c = dict(logits=logits, tokens=tokens, uniforms=torch.rand(B, T, generator=gen), parents=parents)
    p = torch.softmax(logits[0, 0].double(), -1)
    for probs in (near, None):
        paths, counts, following = run(dict(c, draft_probs=probs))
        second = paths[:, 1].long().clamp(min=0).cpu()
        first = torch.where(counts.cpu() > 1, tokens.gather(1, second[:, None])[:, 0], following.cpu())
        if probs is None:  # certain drafts: exact for any fixed tree
            tokens_one = tokens[:1].expand(B, T)
            paths, counts, following = run(dict(c, tokens=tokens_one, draft_probs=None))
            second = paths[:, 1].long().clamp(min=0).cpu()
            first = torch.where(counts.cpu() > 1, tokens_one.gather(1, second[:, None])[:, 0], following.cpu())
        seen = torch.bincount(first, minlength=V).double() / B
        assert ((seen - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all()


def test_rows_without_a_distribution():
    c = case(5, 3, 100, "chain", True)
    c["uniforms"][:, 1:] = 0.0  # whatever is likely at all is kept
    c["logits"][0, 0, 5] = float("nan")
    c["logits"][1, 1, 7] = float("inf")
    c["logits"][2, 0] = float("-inf")
    c["logits"][3, 0, 50:] = float("-inf")
    c["tokens"][3, 1] = 70  # no weight: refused
    want = check(c)
    assert want[2][0] == -1 and want[1][0] == 1 and want[2][1] == -1 and want[1][1] == 2
    assert want[2][2] == -1 and want[1][3] == 1
    check(dict(c, draft_probs=None))
    check(c, 0.0)


def test_draft_probabilities_that_are_odd():
    c = case(6, 5, 64, "star", True)
    c["draft_probs"] = c["draft_probs"].clone()
    c["draft_probs"][0, 0, :8] = float("nan")
    c["draft_probs"][1, 0] = -1.0
    c["draft_probs"][2, 0] = 5.0          # nothing is left: the distribution stays
    c["draft_probs"][3, 0] = torch.softmax(c["logits"][3, 0], -1)  # the target's own
    c["uniforms"][:, 1:] = 0.999
    check(c)
    for t in (torch.bfloat16, torch.float16):
        check(dict(c, draft_probs=c["draft_probs"].to(t)))


def test_layouts_types_and_streams():
    c = case(4, 6, 1003, "tree", True)
    want = [x.cpu() for x in run(c)]
    wide = torch.zeros(4, 9, 1010)
    wide[:, 2:8, 3:1006] = c["logits"]
    probs = torch.zeros(5, 4, 2000)
    probs[:, :, 1:1004] = c["draft_probs"].transpose(0, 1)
    other = dict(logits=wide.to(DEV)[:, 2:8, 3:1006], draft_probs=probs.to(DEV).transpose(0, 1)[:, :, 1:1004],
                 tokens=c["tokens"].int().to(DEV), uniforms=c["uniforms"].to(DEV),
                 parents=torch.cat([c["parents"]] * 2, 1).to(DEV)[:, :6])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b2.b200_verify_drafts(**other)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x.cpu(), y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = b2.b200_verify_drafts(**other)
    other["uniforms"].copy_(torch.rand(4, 6))
    graph.replay()
    again = b2.b200_verify_drafts(**other)
    assert all(torch.equal(x, y) for x, y in zip(out, again))


def test_bad_numbers_are_reported():
    c = case(3, 5, 100, "chain", True)
    c["uniforms"][:, 1:] = 0.0
    good = run(c)

    def reported(**kw):
        clear_device_errors(DEV)
        on = {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in dict(c, **kw).items()}
        out = b2.b200_verify_drafts(**on)
        torch.cuda.synchronize()
        assert read_device_errors(DEV)
        clear_device_errors(DEV)
        return out

    tokens = c["tokens"].clone()
    tokens[1, 2], tokens[2, 1] = 100, -1
    paths, counts, following = reported(tokens=tokens)
    assert torch.equal(paths[0], good[0][0]) and int(counts[1]) == 2 and int(counts[2]) == 1
    assert (following >= 0).all()
    parents = torch.tensor([-1, 0, 2, 7, -2], dtype=torch.int32)
    assert reported(parents=parents)[1].tolist() == [2, 2, 2]
    paths, counts, following = reported(draft_lens=torch.tensor([5, 6, -1], dtype=torch.int32))
    assert counts.tolist() == [int(good[1][0]), 0, 0] and following[1:].tolist() == [-1, -1]
