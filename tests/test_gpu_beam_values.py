"""Beam selection's sums and merge, at the rows where they go wrong first."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def plain_select(logits, scores, n):
    """Values, parents and tokens in float64, differences ahead of sums: value = score + ((x - max) - log sum exp(x - max))."""
    B, K = scores.shape
    x = logits.double().cpu().numpy().reshape(B, K, -1)
    s = scores.double().cpu().numpy()
    V = x.shape[-1]
    val = np.full((B, K, V), -np.inf)
    for b in range(B):
        for k in range(K):
            top = x[b, k].max()
            if s[b, k] > -np.inf and np.isfinite(top):
                d = x[b, k] - top
                val[b, k] = s[b, k] + (d - np.log(np.exp(d).sum()))
    flat = val.reshape(B, -1)
    at = np.argsort(-flat, axis=1, kind="stable")[:, :n]
    return np.take_along_axis(flat, at, 1), at // V + np.arange(B)[:, None] * K, at % V


def check(logits, scores, n, atol, strict=False):
    """Values within atol and their own rounding (2^-24); the same continuations, unless (strict: not even then) two of different rows lie closer together
    than that."""
    from transformer_surgeon_b200 import ops
    total = logits.numel() // scores.shape[0]
    val, parents, tokens = plain_select(logits, scores, min(n + 1, total))
    got = [o.cpu().numpy() for o in ops.beam_select(logits, scores, n)]
    alive = np.isfinite(val[:, :n])
    assert (np.isfinite(got[0]) == alive).all()
    err = np.abs(np.where(alive, got[0] - np.where(alive, val[:, :n], 0), 0))
    assert (err <= atol + 2.0 ** -24 * np.abs(np.where(alive, val[:, :n], 0))).all(), err.max()
    for b, i in zip(*np.nonzero((got[1] != parents[:, :n]) | (got[2] != tokens[:, :n]))):
        near = [j for j in range(val.shape[1]) if parents[b, j] != parents[b, i] and abs(val[b, j] - val[b, i]) <= 2 * atol]
        assert near and not strict, (b, i, got[1][b], parents[b], got[2][b], tokens[b])


# A dominating term, the last one of its thread: its argument x log2 e - R, at most 4 above, is rounded once (2^-23 bits: 8.3e-8 of the term), its exponential
# is off by 2^-22 (2.4e-7), two additions follow or precede it (2^-24 each): 4.4e-7 of the sum, hence of the logarithm.
@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("above", [2, 12, 25, 45, 65, 200])
def test_a_late_peak_keeps_its_bits(cuda, name, above):
    K, V, n = 16, 40000, 32                        # two stretches a row, of several tiles each
    g = torch.Generator().manual_seed(above)
    x = torch.randn(K, V, generator=g)
    x[:, -1] = 4 + above + torch.rand(K, generator=g)
    scores = -0.25 * torch.arange(K).float()[None]
    check(x.to(DT[name]).to(cuda), scores.to(cuda), n, 4.6e-7 if above > 2 else 5.5e-6)


# Sums of at most 80 terms a thread, in fp32: 80 * 2^-24 and the above, 5.3e-6 at worst.
@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(16, 40000, 32), (3, 40000, 8)])
@pytest.mark.parametrize("kind", ["-1e9", "-1e10", "-1e30", "-1e37", "-3e38", "1e10", "3e38", "about 1e8", "about 1e10", "about -1e10", "edge", "-edge", "late peak of 1e10",
                                  "late ones in a mask of -1e10", "late ones in a mask of -1e30", "late ones in a mask of the lowest value", "mask of -1e30 and -inf",
                                  "two masks", "late 3e38"])
def test_logits_of_any_size(cuda, name, shape, kind):
    """Masks of large negative numbers, whole rows of them among these, and logits as large as the type holds: every finite logit counts."""
    K, V, n = shape
    g = torch.Generator().manual_seed(7)
    x = torch.randn(K, V, generator=g)
    late = torch.arange(V) >= V - 100
    if kind == "about 1e8":
        x = 1e8 + 8 * x.round()
    elif kind in ("about 1e10", "about -1e10"):
        x = float(kind.split()[1]) * (1 + 1e-6 * x)
    elif kind in ("edge", "-edge"):                # 2^22 / log2 e = 2907270
        x = (2907270 + x) * (1 if kind == "edge" else -1)
    elif kind == "late peak of 1e10":
        x[:, -5] = 1e10
    elif kind.startswith("late ones"):
        low = {"-1e10": -1e10, "-1e30": -1e30, "value": torch.finfo(DT[name]).min}[kind.split()[-1]]
        x = torch.where(late, x, torch.tensor(low))
    elif kind == "mask of -1e30 and -inf":
        x = torch.where(torch.arange(V) % 3 == 0, torch.tensor(-1e30), torch.tensor(float("-inf"))).expand(K, V)
    elif kind == "two masks":
        x = torch.where(torch.arange(V) % 1000 == 999, torch.tensor(-1e30), torch.tensor(torch.finfo(DT[name]).min)).expand(K, V)
    elif kind == "late 3e38":
        x[:, -3:] = 3e38
    else:
        x = torch.full((K, V), float(kind))
    scores = -0.25 * torch.arange(K).float()[None]
    check(x.to(DT[name]).to(cuda), scores.to(cuda), n, 5.5e-6)


@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_infinite_and_missing_logits_beside_large_ones(cuda, name):
    """A NaN or +infinity takes a row out, wherever it stands among logits of any size; -infinity does not."""
    from transformer_surgeon_b200 import ops
    K, V = 8, 40000
    x = torch.randn(K, V, generator=torch.Generator().manual_seed(3))
    x[1], x[2, -7], x[3] = -1e30, float("inf"), 1e10
    x[3, 9] = float("nan")
    x[4] = float("nan")
    x[5], x[5, 20000] = -1e10, float("inf")
    x[6] = float("-inf")
    x[7] = float("-inf")
    x[7, -1] = -1e30
    x[1, 5] = float("-inf")
    scores = torch.zeros(1, K)
    v, p, t = (o.cpu() for o in ops.beam_select(x.to(DT[name]).to(cuda), scores.to(cuda), 32))
    assert v.isfinite().all() and set(p[0].tolist()) <= {0, 1, 7}
    assert (p[0, 0], t[0, 0], v[0, 0]) == (7, V - 1, 0.0)          # the only one of its row
    dead = x.clone()
    dead[[0, 1, 7]] = float("nan")
    v, p, t = (o.cpu() for o in ops.beam_select(dead.to(DT[name]).to(cuda), scores.to(cuda), 5))
    assert (v == float("-inf")).all() and t[0].tolist() == [0, 1, 2, 3, 4]


@pytest.mark.parametrize("K,n,kind", [(40, 32, "one value"), (256, 5, "one value"), (256, 32, "one value"), (40, 32, "some rows out"), (64, 32, "few values"),
                                      (40, 32, "unequal scores"), (120, 9, "some rows out")])
def test_merge_of_more_equal_entries_than_it_has_room_for(cuda, K, n, kind):
    """K * n entries, all or most of them at the n-th value: the lowest k * V + t stay."""
    V = 3000
    x = torch.full((K, V), 1.5)
    scores = torch.zeros(2, K)
    if kind == "some rows out":
        scores[:, 3::7] = float("-inf")
    elif kind == "few values":
        x = torch.randint(0, 2, (K, V), generator=torch.Generator().manual_seed(1)).float()[:1].expand(K, V)
    elif kind == "unequal scores":
        scores[0, ::2] = -1.0
    check(torch.cat((x, x.flip(1))).contiguous().to(cuda), scores.to(cuda), n, 2e-6, strict=True)             # rows are equal bit by bit, so are their sums
