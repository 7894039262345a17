"""Decode attention over pages with their own scales: the choice between whole and cut sequences, and the bits that scores and weights keep."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


@pytest.mark.parametrize("B,L,H,hkv,d,name,cut", [(40, 600, 14, 2, 64, "fp32", False), (100, 1000, 14, 2, 64, "fp32", True), (50, 900, 28, 4, 128, "fp32", True),
                                                  (60, 700, 24, 2, 128, "bf16", False), (30, 2000, 24, 2, 128, "bf16", True), (4, 519, 14, 2, 64, "bf16", True),
                                                  (58, 575, 32, 8, 128, "bf16", False)])
def test_sequences_are_cut_by_the_ctas_that_the_launch_has(cuda, B, L, H, hkv, d, name, cut):
    """A kv head's query heads may take several CTAs (8 of bf16, 4 of fp32 each), which leaves fewer ranges.  Parts of cut sequences are what the
    workspace is written for."""
    from tests.test_gpu_beams import make_kv
    from transformer_surgeon_b200 import ops
    kv = make_kv(B, (L + 15) // 16, hkv, d, cuda, lens=[L] * B)
    ws = torch.zeros(ops.decode_attn_workspace_bytes(B, H, d, L), dtype=torch.uint8, device=cuda)
    ops.paged_decode_attention(kv, torch.ones(B, H, d, dtype=DT[name], device=cuda), L, ws=ws)
    assert bool(ws[ops.COUNTER_BYTES:].any()) == cut


def error_bound(name, s, exponents, size, ref):
    """|out - exact| for scores that are single products, s [.., tokens] in nats of 40 tokens at most.
    A score: its query is two f16 terms (2^-22) or a bf16 number, its factor is rounded three times, 2^-24 each, and holds log2 e to 2^-25; in bits it is added to V's exponent and taken
    from M, at most 14 bits above, each rounded by 2^-24 of what comes out.  A weight: exponential 2^-22, two f16 terms 2^-22 or (bf16) one, 2^-11.  The sums: three MMAs of 16 products and
    an accumulator, each addend cut at 2^-23 of the largest; the denominator's sums, the quotient and the output 2^-20.  Score errors count in numerator and denominator.  The
    output of bf16 is rounded by 2^-8."""
    top = np.abs(s).max(-1)
    score = top * (2.0 ** -22 + 4 * 2.0 ** -24) + np.log(2) * 2.0 ** -24 * (3 * top / np.log(2) + 2 * np.abs(exponents).max() + 30)
    share = 2 * score + 3 * 2.0 ** -22 + 3 * 17 * 2.0 ** -23 + 2.0 ** -20
    if name == "bf16":
        return (share + 2.0 ** -11)[..., None] * size + 2.0 ** -8 * np.abs(ref)
    return share[..., None] * size


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("d,hkv,g", [(128, 2, 4), (64, 2, 7), (128, 1, 1), (64, 1, 12)])
def test_scores_and_weights_keep_their_bits(cuda, name, d, hkv, g):
    """Keys and queries with one element each that is not zero: scores are single products, so that what queries, weights and sums lose shows.  fp32 with one f16 term for
    the weights, or for the queries, would be outside of the bound."""
    from tests.test_gpu_beams import Plain, make_kv, plain_attention
    from transformer_surgeon_b200 import ops
    lens, H = [40, 33, 16, 5], hkv * g
    B, T = len(lens), max(lens)
    kv = make_kv(B, 3, hkv, d, cuda, lens=lens)
    gen = torch.Generator().manual_seed(d + g)
    k, q, at = torch.zeros(B, T, hkv, d), torch.zeros(B, H, d), 5 * torch.arange(hkv) + 3
    for h in range(hkv):
        k[:, :, h, at[h]] = 8 * torch.rand(B, T, generator=gen) - 4
        q[:, h * g:(h + 1) * g, at[h]] = 1 + torch.rand(B, g, generator=gen)
    q = q.to(DT[name])
    kv.append(k.to(cuda), torch.randn(B, T, hkv, d, generator=gen).to(cuda), seq_lens=torch.zeros_like(kv.seq_lens))
    out = ops.paged_decode_attention(kv, q.to(cuda), 48, sm_scale=1.0).double().cpu().numpy()
    ref, size = plain_attention(kv, q, lens, 1.0)
    p, table = Plain(kv), kv.block_table.cpu().numpy()
    short = {"weights": False, "queries": False}
    for b, n in enumerate(lens):
        ids = table[b, :(n + 15) // 16]
        for h in range(H):
            kk, vv = (x[ids, h // g].reshape(-1, d)[:n] for x in (p.k, p.v))
            x = q[b, h].double().numpy()
            s = kk @ x
            bound = error_bound(name, s[None], np.log2(p.vs[ids, h // g]), size[b, h][None], ref[b, h][None])[0]
            assert (np.abs(out[b, h] - ref[b, h]) <= bound).all(), (np.abs(out[b, h] - ref[b, h]) / bound).max()
            w = np.exp(s - s.max())
            short["weights"] |= bool((np.abs(w.astype(np.float16).astype(np.float64) @ vv / w.sum() - ref[b, h]) > bound).any())
            w1 = np.exp(kk @ x.astype(np.float16).astype(np.float64))
            short["queries"] |= bool((np.abs(w1 @ vv / w1.sum() - ref[b, h]) > bound).any())
    assert name == "bf16" or (short["weights"] and short["queries"])
