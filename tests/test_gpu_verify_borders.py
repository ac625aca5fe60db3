"""q3_verify_drafts where the drawn token lies at the borders of a row's pieces: its first and last tokens,
those around every border that a cut among CTAs and warps may have, and vocabularies that leave warps without
a piece or are no multiple of 4."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import torch
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch


def border_tokens(vocab, most=600):
    """The row's ends, and the tokens around the borders of its pieces and of the pieces' pieces."""
    at = set(range(min(vocab, 9))) | set(range(max(0, vocab - most), vocab))
    for ctas in (1, 2, 4, 8, 16):
        for warps in (8, 16):
            per = -(-(-(-vocab // (ctas * warps))) // 4) * 4
            borders = list(range(0, vocab, per * warps)) + [x for x in range(0, vocab, per)][-3:]
            last = (vocab - 1) // per * per
            sub = -(-(-(-min(per, vocab - last) // warps)) // 4) * 4
            borders += list(range(last, vocab, sub))
            at |= {b + o for b in borders for o in (-5, -4, -1, 0, 1, 3, 4)}
    return sorted(t for t in at if 0 <= t < vocab)


def draw(T, q3, target, draft, n_seqs, vocab, width, us):
    """The tokens drawn from rows [n, width] of `target` (less `draft`'s, whose drafted token 0 is rejected),
    n_seqs rows a call."""
    n = target.shape[0]
    k = 0 if draft is None else 1
    out = T.full((n, k + 1), -7, dtype=T.int32, device="cuda")
    acc = T.full((n,), -7, dtype=T.int32, device="cuda")
    toks = T.zeros(n, max(k, 1), dtype=T.int32, device="cuda")
    ua = T.ones(n, max(k, 1), device="cuda")
    for i in range(0, n, n_seqs):
        q3.verify_drafts(out[i].data_ptr(), acc[i:].data_ptr(), target[i].data_ptr(), width, width,
                         draft[i].data_ptr() if k else None, width, width,
                         toks[i].data_ptr() if k else None, None, ua[i].data_ptr() if k else None,
                         us[i:].data_ptr(), min(n_seqs, n - i), k, vocab)
    T.cuda.synchronize()
    assert bool((acc == 0).all())
    return out[:, 0].tolist()


VOCABS = [151936, 128256, 129280, 81000, 81001, 50257, 50259, 16385, 8192, 8193, 4095, 700, 129, 128, 5, 1]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("n_seqs", [1, 4, 8, 64])
@pytest.mark.parametrize("pad", [0, 3])
def test_one_hot_rows(T, q3lib, vocab, n_seqs, pad):
    """All of a row's mass on one token: that token, for whatever number in [0, 1). Rows on 16-byte
    boundaries (their width rounded up to a multiple of 4), and 3 values wider, which shifts them."""
    width = -(-vocab // 4) * 4 + pad
    tokens = border_tokens(vocab, most=600 if n_seqs == 1 else 150)
    got, rest = [], tokens
    while rest:
        here, rest = rest[:256], rest[256:]
        target = T.full((len(here), width), 9.0, device="cuda")
        target[:, :vocab] = 0.0
        target[T.arange(len(here)), T.tensor(here)] = 0.75
        us = T.tensor([(0.0, 0.37, 1 - 2.0 ** -24)[i % 3] for i in range(len(here))], device="cuda")
        got += draw(T, q3lib, target, None, n_seqs, vocab, width, us)
    assert got == tokens


@pytest.mark.parametrize("vocab", [151936, 81001, 81000, 50257, 8193])
@pytest.mark.parametrize("n_seqs", [1, 8])
def test_one_hot_residuals(T, q3lib, vocab, n_seqs):
    """The same of target less draft, both rows aligned: the draft's mass lies on token 0, which is rejected
    (target 0 there), and half of the target's on the border token."""
    width = -(-vocab // 4) * 4
    tokens = [t for t in border_tokens(vocab, most=200) if t > 1][-256:]
    target = T.zeros(len(tokens), width, device="cuda")
    target[T.arange(len(tokens)), T.tensor(tokens)] = 0.5
    target[:, 1] = 0.25
    draft = T.zeros_like(target)
    draft[:, 0], draft[:, 1] = 0.5, 0.25
    us = T.rand(len(tokens), device="cuda")
    assert draw(T, q3lib, target, draft, n_seqs, vocab, width, us) == tokens


@pytest.mark.parametrize("vocab", [151936, 128256, 81001, 50257, 8193, 300])
@pytest.mark.parametrize("n_seqs", [1, 4, 8, 64])
def test_either_side_of_a_border(T, q3lib, vocab, n_seqs):
    """Four tokens of a quarter each around a border: C passes u * C_last at the token whose share holds u,
    and u on a border belongs to the token behind it. Quarters add up exactly in any order."""
    width = -(-vocab // 4) * 4
    tokens = [t for t in border_tokens(vocab, most=40) if 4 <= t < vocab - 1][-120:]
    target = T.zeros(len(tokens), width, device="cuda")
    rows, want, us = T.arange(len(tokens)), [], []
    at = T.tensor([[0, t - 1, t, vocab - 1] for t in tokens])
    for j in range(4):
        target[rows, at[:, j]] = 0.25
    for i in range(len(tokens)):
        j = i % 4
        us.append((j * 0.25, j * 0.25 + 0.25 - 2.0 ** -24)[i // 4 % 2])
        want.append(int(at[i, j]))
    assert draw(T, q3lib, target, None, n_seqs, vocab, width, T.tensor(us, device="cuda")) == want
