"""The likeliest tokens where fp32 logits do not tell them apart: low temperatures, large hidden states,
more near ties than a few tiles hold; logits that are not finite; a vocabulary of more than 2^27 tokens."""
import pytest
import torch

import grad_ref as R
from fastmlx_amd import ops
from gpu_util import announce
from test_gpu_logprobs import case, check_scores

pytestmark = pytest.mark.gpu

ROWS = [10, 60, 300, 1800]  # one for each product


def copies(gpu, M, V, K, n, small, seed=1):
    """n tokens whose weights are one row's but for scales of four groups, where h is `small` of its size
    elsewhere: their logits differ by less than fp32 sums of the whole row see."""
    h, w, W, ids, gen = case(gpu, M, V, K, 1, seed=seed)
    words, s, b = (t.clone() for t in w)
    at = torch.randperm(V, generator=gen)[:n].to(gpu)
    words[at], s[at], b[at] = w[0][0], w[1][0], w[2][0]
    s[at, :4] = (s[at, :4].float() * (0.5 + torch.rand(n, 4, generator=gen).to(gpu))).bfloat16()
    h[:] = (W[0] * (0.5 + 0.01 * torch.randn(M, 1, generator=gen).to(gpu))).bfloat16()
    h[:, :256] *= small
    w = (words, s, b)
    return h, w, R.values(*w, 4, 64), ids


def falling(got):
    assert bool((got[4][:, 1:] <= got[4][:, :-1]).all()), "top_logp falls"


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("T", [1.0, 1e-4, 1e-7])
def test_near_ties_at_low_temperatures(gpu, M, T):
    announce(f"near ties {M} {T}")
    h, w, W, ids = copies(gpu, M, 4000, 512, 60, 1e-7)
    got, _ = check_scores(h, w, W, ids, 50, T=T)
    falling(got)


@pytest.mark.parametrize("M", ROWS)
def test_near_ties_of_large_hidden_states(gpu, M):
    announce(f"near ties of large states {M}")
    h, w, W, ids = copies(gpu, M, 4000, 512, 60, 1e-7, seed=2)
    got, _ = check_scores((h.float() * 2.0 ** 17).bfloat16(), w, W, ids, 50)
    falling(got)


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("top", [1, 20, 64])
def test_near_ties_in_every_tile(gpu, M, top):
    """More of them than there are tiles: their exact order decides, whatever their tiles' largest."""
    announce(f"near ties in every tile {M} {top}")
    h, w, W, ids = copies(gpu, M, 40000, 512, 3000, 1e-7, seed=3)
    got, _ = check_scores(h, w, W, ids, top)
    falling(got)


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("V", [4, 50])
def test_tokens_alike_to_fp32(gpu, M, V):
    """All logits the same in fp32, none in 64 bits."""
    announce(f"alike to fp32 {M} {V}")
    h, w, W, ids = copies(gpu, M, V, 512, V, 1e-10, seed=4)
    got, _ = check_scores(h, w, W, ids, V)
    falling(got)


@pytest.mark.parametrize("M", ROWS)
def test_weights_of_zeros(gpu, M):
    """A head of zeros, for any hidden state: all logits are 0, and the lower tokens come first."""
    V = 3000
    announce(f"zeros {M}")
    h, w, W, ids, _ = case(gpu, M, V, 128, 1)
    w = (w[0], torch.zeros_like(w[1]), torch.zeros_like(w[2]))
    got = ops.head_logprobs(h, *w, ids, top=40)
    assert torch.equal(got[3].long(), torch.arange(40, device=gpu).expand(M, 40))
    flat = torch.log(torch.tensor(float(V), dtype=torch.float64, device=gpu))
    for t in (got[1], got[2], -got[4]):
        R.check(t, flat.expand(t.shape), (flat * 4 * R.U32).expand(t.shape), "flat")


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("V", [3000, 37])
def test_a_logit_of_minus_infinity(gpu, M, V):
    """One such logit makes its row's numbers NaN, whatever else is in its tile."""
    announce(f"minus infinity {M} {V}")
    h, (words, s, b), W, ids, _ = case(gpu, M, V, 128, 2, absent=0.0)
    h[:, :64] = h[:, :64].abs() + 0.125
    b[V // 2, 0] = float("-inf")
    got = ops.head_logprobs(h, words, s, b, ids, top=9)
    for i in (0, 1, 2, 4):
        assert got[i].isnan().all(), i
    assert bool((got[3] == -1).all())
    a = torch.ones(M, 2, device=gpu)
    assert ops.head_logprobs_grad(h, words, s, b, ids, *got[:3], a).isnan().all()


@pytest.mark.parametrize("M", [1, 4, 5])
def test_a_vocabulary_beyond_the_few_row_products_blocks(gpu, M):
    """2^27 tokens and more, of which a few have weights other than zero."""
    V, K = 2 ** 27 + 5000, 32
    announce(f"{V} tokens, {M} rows")
    words = torch.zeros(V, K // 8, dtype=torch.int32, device=gpu)
    s, b = (torch.zeros(V, 1, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    gen = torch.Generator().manual_seed(5)
    at = torch.tensor([0, 17, 2 ** 26, 2 ** 27 - 1, 2 ** 27 + 4096, V - 1], device=gpu)
    b[at, 0] = torch.tensor([1.0, 3.0, -2.0, 2.5, 3.5, 2.0], device=gpu).bfloat16()
    h = torch.rand(M, K, generator=gen).bfloat16().to(gpu)
    ids = at[torch.arange(M, device=gpu) % 6][:, None].int()
    got = ops.head_logprobs(h, words, s, b, ids, top=3, group_size=32)
    l = h.double().sum(-1, keepdim=True) * b[at, 0].double()
    lse = torch.log(V - 6 + l.exp().sum(-1))
    # Sums of 2^27 terms of 1: each thread's and the tiles' in fp32, a few thousand one after another.
    tol = 2.0 ** -10 + 0 * lse
    R.check(got[2], lse, tol, "lse")
    R.check(got[0][:, 0], l.gather(1, (torch.arange(M, device=gpu) % 6)[:, None])[:, 0] - lse, tol, "logp")
    assert torch.equal(got[3].long(), at[[4, 1, 3]].expand(M, 3))


@pytest.mark.parametrize("M", ROWS)
@pytest.mark.parametrize("V", [3, 5000])
@pytest.mark.parametrize("T", [1.0, 1e-6])
@pytest.mark.parametrize("part", [1, 3])
def test_a_likeliest_token_that_fp32_rounds(gpu, M, V, T, part):
    """The likeliest token's logit 8.5 + part / 32 as 2^20 + 8.5 + part / 32 - 2^20, which fp32 rounds (down for 1, up
    for 3); the others' is 8 exactly: what its sum is off by reaches other tokens' numbers by its probability only,
    and its own by what the others have.  At the low temperature it is off by thousands, and the others have nothing."""
    announce(f"rounded leader {M} {V} {T} {part}")
    K = 512
    words = torch.zeros(V, K // 8, dtype=torch.int32, device=gpu)
    s = torch.zeros(V, K // 64, dtype=torch.bfloat16, device=gpu)  # all weights of a group are its bias
    b = torch.zeros_like(s)
    b[:, 0] = 8.0
    lead = V // 2
    b[lead] = torch.tensor([2.0 ** 20, 0, 0, 8.5, part / 32, 0, 0, -2.0 ** 20], device=gpu).bfloat16()
    h = torch.zeros(M, K, dtype=torch.bfloat16, device=gpu)
    h[:, ::64] = 1.0
    ids = torch.tensor([[0, lead]], dtype=torch.int32, device=gpu).expand(M, 2).contiguous()
    got = ops.head_logprobs(h, words, s, b, ids, top=2, temperature=T)
    l = torch.full((V,), 8.0 / T, dtype=torch.float64, device=gpu)
    l[lead] = (8.5 + part / 32) / T
    lse = torch.logsumexp(l, -1)
    p = float((l[lead] - lse).exp())
    # Of the leader 8 products of 2^20 at most, of the others the scaling to units of log 2 and back; two logarithms.
    el = (10 * R.U32 * 2 ** 21 + 8 * R.U32 * 8) / T
    tol = torch.tensor([p * el, (1 - p) * (8 * R.U32 * 8 / T + 16 * R.U32)], dtype=torch.float64, device=gpu)
    want = l[ids.long()] - lse
    R.check(got[0], want, tol + 32 * R.U32 * (1 + want.abs()), "logp")
    assert bool((got[3] == torch.tensor([lead, 0], dtype=torch.int32, device=gpu)).all())
    assert torch.equal(got[4], got[0].flip(1))
