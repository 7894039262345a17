"""Beam search over 8-bit pages with their own scales: append, decode attention, selection and reordering against plain forms in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
PAGE = 16


def e4m3(x):
    """Nearest e4m3 value, ties to even, saturating (float64)."""
    x = np.clip(x, -448, 448)
    _, e = np.frexp(np.abs(x))
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(x / step) * step


def page_scale(amax):
    """Smallest power of two s, 2^-40 <= s <= 2^40, with amax <= 448 s."""
    m, e = np.frexp(np.asarray(amax, dtype=np.float64))
    return np.exp2(np.clip(np.where(amax > 0, e - 9 + (m > 0.875), -40), -40, 40).astype(np.float64))


def decode(pool, side, d):
    """uint8 [pages, hkv, record] -> values without scale [pages, hkv, 16, d] and scales [pages, hkv], float64."""
    codes = pool[..., :PAGE * d].contiguous().view(torch.float8_e4m3fn).float().double().cpu().numpy()
    codes = codes.reshape(*codes.shape[:2], PAGE, d) if side == 0 else codes.reshape(*codes.shape[:2], d, PAGE).swapaxes(2, 3)
    return codes, pool[..., PAGE * d:PAGE * d + 4].contiguous().view(torch.float32)[..., 0].double().cpu().numpy()


def make_kv(B, pages, hkv, d, dev, seed=0, lens=None):
    from transformer_surgeon_b200 import ops
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * pages + 2, generator=g)[:B * pages].to(torch.int32).reshape(B, pages).to(dev)
    seq = torch.tensor(lens if lens is not None else [0] * B, dtype=torch.int32, device=dev)
    return ops.PagedKV("fp8_page", B * pages + 2, hkv, d, table, seq, dev)


def fill(kv, n, seed, dtype=torch.float32, spread=None):
    """Appends n tokens of N(0, 1) (times spread [n] per token) to every sequence, from position 0, in one call."""
    B = kv.block_table.shape[0]
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, B, n, kv.hkv, kv.head_dim, generator=g)
    if spread is not None:
        x = x * spread[None, None, :, None, None]
    x = x.to(dtype).to(kv.k_pool.device)
    kv.append(x[0], x[1], seq_lens=torch.zeros_like(kv.seq_lens))
    return x


def rope_tables(d, n, dev):
    a = torch.arange(n, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, d, 2).double() / d)
    return a.cos().float().to(dev), a.sin().float().to(dev)


class Plain:
    """The cache's pages in 64 bits: values, scales."""

    def __init__(self, kv):
        d = kv.head_dim
        (self.k, self.ks), (self.v, self.vs) = decode(kv.k_pool, 0, d), decode(kv.v_pool, 1, d)
        self.k, self.v = self.k * self.ks[..., None, None], self.v * self.vs[..., None, None]

    def append(self, kv, k, v, lens, counts):
        """k, v float64 [B, T, hkv, d] (rotated already): what the pages must hold afterwards."""
        table = kv.block_table.cpu().numpy()
        for b in range(len(lens)):
            at, left = int(lens[b]), int(counts[b])
            j = 0
            while left > 0:
                c = at % PAGE
                n = min(left, PAGE - c)
                if at // PAGE < table.shape[1]:
                    p = table[b, at // PAGE]
                    for vals, scales, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
                        new = x[b, j:j + n].swapaxes(0, 1)                                  # [hkv, n, d]
                        s = page_scale(np.where(np.isfinite(new), np.abs(new), 0).max((1, 2)))
                        s = np.maximum(s, scales[p]) if c else s
                        old = e4m3(vals[p, :, :c] / s[:, None, None]) * s[:, None, None]
                        vals[p] = 0
                        vals[p, :, :c] = old
                        vals[p, :, c:c + n] = e4m3(new / s[:, None, None]) * s[:, None, None]
                        scales[p] = s
                at, j, left = at + n, j + n, left - n


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("d,hkv,H", [(128, 2, 6), (64, 3, 3)])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 77])
def test_append_without_rotation_is_exact(cuda, name, d, hkv, H, T):
    """Codes, scales and slots behind the end, whatever the position inside a page: equal to the definition in 64 bits, K and V alike."""
    lens = [0, 1, 15, 16, 30, 47]
    counts = [T, T, 0, T, max(T - 1, 0), T]
    B = len(lens)
    kv = make_kv(B, (47 + T + 15) // PAGE + 1, hkv, d, cuda, lens=lens)
    fill(kv, 48, seed=T)
    kv.k_pool[-1] = kv.v_pool[-1] = 7
    want = Plain(kv)
    g = torch.Generator().manual_seed(50 + T)
    # tokens of very different sizes: some raise their page's scale, some do not; zeros too
    x = torch.randn(B, T, 2 * hkv, d, generator=g) * torch.exp2(torch.randint(-8, 9, (B, T, 2 * hkv, 1), generator=g).float())
    x[:, T // 2, 0] = 0
    x = x.to(DT[name]).to(cuda)
    k, v = x[:, :, :hkv], x[:, :, hkv:]                        # strided tokens
    kv.append(k, v, new_lens=torch.tensor(counts, dtype=torch.int32, device=cuda))
    want.append(kv, k.double().cpu().numpy(), v.double().cpu().numpy(), lens, counts)
    got = Plain(kv)
    for a, b in ((got.k, want.k), (got.v, want.v), (got.ks, want.ks), (got.vs, want.vs)):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("d,hkv,H", [(128, 2, 7), (64, 1, 5)])
@pytest.mark.parametrize("T,shift", [(1, 0), (33, 0), (33, 1)])
def test_rope_append(cuda, name, d, hkv, H, T, shift):
    """Rotated keys and queries.  A code is at most half an e4m3 step (2^-4 of the value, 2^-10 of the scale below 2^-6) from the exact rotation and
    2^-22 of its pair's size (two products and a sum in fp32); the query is rounded once more.  shift: tokens that start at odd elements."""
    lens = [3, 40]
    B = 2
    kv = make_kv(B, 8, hkv, d, cuda, lens=lens)
    fill(kv, 40, seed=1)
    cos, sin = rope_tables(d, 128, cuda)
    g = torch.Generator().manual_seed(9)
    width = (H + 2 * hkv) * d + (5 if shift else 0)            # an odd stride: no vector accesses
    buf = (torch.randn(B * T * width + 8, generator=g) * 3).to(DT[name]).to(cuda)[shift:]
    x = buf[:B * T * width].view(B, T, width)
    q, k, v = (x[..., a * d:b * d].unflatten(2, (b - a, d)) for a, b in ((0, H), (H, H + hkv), (H + hkv, H + 2 * hkv)))
    rest = x[..., (H + 2 * hkv) * d:].clone()

    def turned(t):
        z = t.double().cpu().numpy()
        at = np.asarray(lens)[:, None] + np.arange(T)
        c, s = (w.double().cpu().numpy()[at][:, :, None] for w in (cos, sin))
        a, b = z[..., :d // 2], z[..., d // 2:]
        size = np.concatenate([np.hypot(a, b)] * 2, -1)
        return np.concatenate([a * c - b * s, b * c + a * s], -1), size
    (qe, qsize), (ke, ksize) = turned(q), turned(k)
    ve = v.double().cpu().numpy()
    kv.rope_append(q, k, v, (cos, sin))
    half = 2.0 ** -8 if name == "bf16" else 2.0 ** -24          # finfo.eps / 2: bf16 has 7 fraction bits, eps 2^-7
    assert (np.abs(q.double().cpu().numpy() - qe) <= half * 1.01 * np.abs(qe) + 2.0 ** -22 * qsize).all()
    np.testing.assert_array_equal(v.double().cpu().numpy(), ve)
    assert torch.equal(x[..., (H + 2 * hkv) * d:], rest)
    got = Plain(kv)
    table = kv.block_table.cpu().numpy()
    for b in range(B):
        at = lens[b] + np.arange(T)
        kk, ks = got.k[table[b, at // PAGE], :, at % PAGE], got.ks[table[b, at // PAGE]]
        assert (np.abs(kk - ke[b]) <= np.maximum(2.0 ** -4 * np.abs(ke[b]), 2.0 ** -10 * ks[..., None]) * 1.001 + 2.0 ** -22 * ksize[b]).all()
        vv, vs = got.v[table[b, at // PAGE], :, at % PAGE], got.vs[table[b, at // PAGE]]
        np.testing.assert_array_equal(vv, e4m3(ve[b] / vs[..., None]) * vs[..., None])
        for p in np.unique(at // PAGE):                         # the scale: of the page's tokens that are new, or of older ones
            mine = np.abs(ke[b][at // PAGE == p]).max((0, 2))
            assert (got.ks[table[b, p]] * 448 >= mine * (1 - 2.0 ** -22)).all()


def test_append_special_values_and_bounds(cuda):
    """Infinite elements saturate and set no scale, NaN stays one, huge and tiny values meet the range of scales, positions beyond the block table and
    pages out of range are skipped, a zero page has the smallest scale."""
    d, hkv = 128, 1
    kv = make_kv(4, 2, hkv, d, cuda, lens=[0, 0, 0, 30])
    x = torch.ones(4, 4, hkv, d, device=cuda)
    x[0, 0, 0, 0], x[0, 1, 0, 1], x[0, 2, 0, 2] = float("inf"), float("-inf"), float("nan")
    x[1] = 0
    x[2, 0], x[2, 1] = 1e30, 1e-30
    v = x.clone()
    kv.append(x, v)
    got = Plain(kv)
    table = kv.block_table.cpu().numpy()
    s = 2.0 ** -8                                               # 1 <= 448 * 2^-8 = 1.75
    for vals, scales in ((got.k, got.ks), (got.v, got.vs)):
        a = vals[table[0, 0], 0]
        assert scales[table[0, 0], 0] == s and a[0, 0] == 448 * s and a[1, 1] == -448 * s and np.isnan(a[2, 2])
        assert np.isnan(a).sum() == 1 and a[3, 3] == 1 and (a[4:] == 0).all()
        assert scales[table[1, 0], 0] == 2.0 ** -40 and (vals[table[1, 0]] == 0).all()
        assert scales[table[2, 0], 0] == 2.0 ** 40 and (vals[table[2, 0], 0, 0] == 448 * 2.0 ** 40).all() and (vals[table[2, 0], 0, 1] == 0).all()
        assert (vals[table[3, 1], 0, 14:] == 1).all()            # two of the four fit
    untouched = kv.k_pool.clone(), kv.v_pool.clone()
    kv.block_table[:] = torch.tensor([-1, kv.num_pages], dtype=torch.int32, device=cuda)
    kv.append(x, v)
    kv.append(x, v, new_lens=torch.zeros(4, dtype=torch.int32, device=cuda))
    kv.append(x, v, seq_lens=torch.full((4,), 1000, dtype=torch.int32, device=cuda))
    kv.append(x[:, :0], v[:, :0])
    assert torch.equal(kv.k_pool, untouched[0]) and torch.equal(kv.v_pool, untouched[1])


def test_append_token_by_token_keeps_what_a_chunk_gives(cuda):
    """Tokens in ascending size one by one: every growth of the scale re-encodes the older ones.  Against the chunk (encoded once) a value may be off by the
    subnormal steps it went through: the last scale's 2^-10 and less for each smaller one, 2^-9 together."""
    kv, one = (make_kv(1, 2, 2, 64, cuda) for _ in range(2))
    spread = torch.exp2(torch.linspace(-6, 6, 20))
    x = fill(kv, 20, 3, spread=spread)
    for t in range(20):
        one.append(x[0, :, t:t + 1], x[1, :, t:t + 1], seq_lens=torch.tensor([t], dtype=torch.int32, device=cuda))
    a, b = Plain(kv), Plain(one)
    table, order = kv.block_table[0].cpu().numpy(), one.block_table[0].cpu().numpy()
    for va, sa, vb, sb in ((a.k, a.ks, b.k, b.ks), (a.v, a.vs, b.v, b.vs)):
        np.testing.assert_array_equal(sa[table], sb[order])
        assert (np.abs(va[table] - vb[order]) <= sa[table][..., None, None] * 2.0 ** -9 + 2.0 ** -3 * np.abs(va[table]) * (np.abs(va[table]) < sa[table][..., None, None] * 2.0 ** -5)).all()


# ------------------------------------------------------------------------------------------------ attention
def plain_attention(kv, q, lens, sm_scale):
    p, table = Plain(kv), kv.block_table.cpu().numpy()
    B, H, d = q.shape
    q = q.double().cpu().numpy().reshape(B, kv.hkv, H // kv.hkv, d)
    out, size = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        if lens[b] > 0:
            ids = table[b, :(lens[b] + PAGE - 1) // PAGE]
            k, v = (x[ids].swapaxes(0, 1).reshape(kv.hkv, -1, d)[:, :lens[b]] for x in (p.k, p.v))
            s = np.einsum("hgd,hld->hgl", q[b], k) * sm_scale
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            out[b], size[b] = np.einsum("hgl,hld->hgd", w, v), np.einsum("hgl,hld->hgd", w, np.abs(v))
    return out.reshape(B, H, d), size.reshape(B, H, d)


# |out - exact| <= C * sum_t p_t |V_t| + rounding of the output (bf16: 2^-8).  bf16: a weight is two e4m3 terms, each off by at most 2^-4 of
# what it stands for: 2^-8; scores are exact sums of two-term queries, in fp32.  fp32: four terms leave 2^-17 of the largest element of a query behind, times |K| * sqrt(d) in a score of
# up to a few tens: 2^-12; CUDA-core kernel: fp32 throughout, its exponential 2^-21 of a score of up to a hundred.
def tolerance(name, size, ref):
    return (2.0 ** -8 * size + 2.0 ** -8 * np.abs(ref) if name == "bf16" else 2.0 ** -12 * size) + 1e-30


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("d,hkv,g", [(128, 2, 4), (128, 1, 1), (128, 2, 7), (64, 2, 7), (64, 1, 8), (128, 1, 12), (64, 3, 17)])
def test_attention(cuda, name, d, hkv, g):
    from transformer_surgeon_b200 import ops
    lens = [0, 1, 2, 15, 16, 17, 33, 97, 200, 1000, 1023]
    B, H = len(lens), hkv * g
    kv = make_kv(B, 65, hkv, d, cuda, seed=3, lens=lens)
    spread = torch.exp2(torch.randint(-3, 4, (1030,), generator=torch.Generator().manual_seed(4)).float() * 0.5)
    fill(kv, 1030, seed=5, spread=spread)
    kv.block_table[1, 1:] = -5                                  # beyond a sequence's pages nothing is looked up
    kv.block_table[2, 1:] = 1 << 30
    q = torch.randn(B, 2, H, d, generator=torch.Generator().manual_seed(6)).to(DT[name]).to(cuda)[:, 1]         # strided sequences
    ref, size = plain_attention(kv, q, lens, d ** -0.5)
    for simt in (False, True):
        for longest in (1030, 1040):                             # other splits
            out = ops.paged_decode_attention(kv, q, longest, simt=simt).double().cpu().numpy()
            assert (np.abs(out - ref) <= tolerance(name, size, ref)).all(), np.abs(out - ref).max()
    short, size = plain_attention(kv, q, [min(x, 40) for x in lens], 0.3)           # lengths beyond max_seq_len are cut
    out = ops.paged_decode_attention(kv, q, 40, sm_scale=0.3).double().cpu().numpy()
    assert (np.abs(out - short) <= tolerance(name, size, short)).all()


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("B,hkv,g,d,L", [(2, 2, 4, 128, 9000), (1, 1, 7, 64, 20011), (40, 8, 4, 128, 500)])
def test_attention_many_splits(cuda, name, B, hkv, g, d, L):
    """Long sequences over many CTAs, and more CTAs than the device holds; twice the same bits."""
    from transformer_surgeon_b200 import ops
    lens = [L - 13 * b for b in range(B)]
    kv = make_kv(B, (L + 15) // 16, hkv, d, cuda, lens=lens)
    fill(kv, L, 8)
    q = torch.randn(B, hkv * g, d, generator=torch.Generator().manual_seed(6)).to(DT[name]).to(cuda)
    ref, size = plain_attention(kv, q, lens, d ** -0.5)
    out = ops.paged_decode_attention(kv, q, L)
    assert (np.abs(out.double().cpu().numpy() - ref) <= tolerance(name, size, ref)).all()
    assert torch.equal(out, ops.paged_decode_attention(kv, q, L))


def test_attention_of_more_sequences_than_a_launch_takes(cuda):
    from transformer_surgeon_b200 import ops
    B, lens = 1100, [(37 * b) % 50 for b in range(1100)]
    kv = make_kv(B, 4, 1, 64, cuda, lens=lens)
    fill(kv, 50, 8)
    q = torch.randn(B, 2, 64, generator=torch.Generator().manual_seed(6)).cuda()
    ref, size = plain_attention(kv, q, lens, 0.125)
    for longest in (50, 64):
        out = ops.paged_decode_attention(kv, q, longest).double().cpu().numpy()
        assert (np.abs(out - ref) <= tolerance("fp32", size, ref)).all()


@pytest.mark.parametrize("B,L", [(2, 3000), (64, 700)])
def test_attention_in_fixed_scratch(cuda, B, L):
    """tsb200_paged_decode_attn_static: cut as far as the library's own scratch has room, whole sequences beyond that."""
    import ctypes as C
    from transformer_surgeon_b200 import _lib, ops
    lens = [L - 7 * b for b in range(B)]
    kv = make_kv(B, (L + 15) // 16, 8, 128, cuda, lens=lens)
    fill(kv, L, 8)
    q = torch.randn(B, 32, 128, generator=torch.Generator().manual_seed(6)).bfloat16().cuda()
    out, desc = torch.empty_like(q), kv.desc()
    for _ in range(2):
        _lib.check(_lib.load().tsb200_paged_decode_attn_static(C.byref(desc), q.data_ptr(), out.data_ptr(), _lib.BF16, 32 * 128, B, 32, 128 ** -0.5, L,
                                                               torch.cuda.current_stream().cuda_stream), "static")
    ref, size = plain_attention(kv, q, lens, 128 ** -0.5)
    assert (np.abs(out.double().cpu().numpy() - ref) <= tolerance("bf16", size, ref)).all()
    assert torch.allclose(out.float(), ops.paged_decode_attention(kv, q, L).float(), rtol=2e-2, atol=2e-2)


def test_attention_on_two_streams(cuda):
    """Two calls at once, each with its own workspace and cache."""
    from transformer_surgeon_b200 import ops
    jobs = []
    for i in range(2):
        lens = [2000 - 300 * i - 11 * b for b in range(6)]
        kv = make_kv(6, 125, 2, 64, cuda, seed=i, lens=lens)
        fill(kv, 2000, 3 + i)
        q = torch.randn(6, 8, 64, generator=torch.Generator().manual_seed(i)).cuda()
        ws = torch.zeros(ops.decode_attn_workspace_bytes(6, 8, 64, 2000), dtype=torch.uint8, device=cuda)
        jobs.append((kv, q, ws, torch.cuda.Stream(), ops.paged_decode_attention(kv, q, 2000, ws=ws).clone()))
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for kv, q, ws, stream, _ in jobs:
            with torch.cuda.stream(stream):
                outs.append(ops.paged_decode_attention(kv, q, 2000, ws=ws))
        torch.cuda.synchronize()
        for out, job in zip(outs, jobs):
            assert torch.equal(out, job[4])


def test_attention_pages_of_extreme_scales(cuda):
    """V scales 2^-40 and 2^40 in one sequence: weights and sums keep every page's share."""
    from transformer_surgeon_b200 import ops
    kv = make_kv(1, 4, 1, 128, cuda, lens=[64])
    fill(kv, 64, 2, spread=torch.cat([torch.full((16,), 2.0 ** e) for e in (-36, 36, -36, 0)]))
    kv.k_pool.zero_()                                            # equal scores
    q = torch.randn(1, 3, 128, device=cuda)
    ref, size = plain_attention(kv, q, [64], 1.0)
    out = ops.paged_decode_attention(kv, q, 64).double().cpu().numpy()
    assert (np.abs(out - ref) <= tolerance("fp32", size, ref)).all()
    kv.v_pool[kv.block_table[0, 1].long()] = kv.v_pool[kv.block_table[0, 0].long()]     # without the large ones: the small ones' own precision
    kv.v_pool[kv.block_table[0, 3].long()] = kv.v_pool[kv.block_table[0, 0].long()]
    ref, size = plain_attention(kv, q, [64], 1.0)
    out = ops.paged_decode_attention(kv, q, 64).double().cpu().numpy()
    assert 0 < np.abs(ref).max() < 2.0 ** -30 and (np.abs(out - ref) <= tolerance("fp32", size, ref)).all()


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_leaves_out_what_is_behind_the_end(cuda, name, d):
    """NaN and infinities cached behind the length that a call gives (tokens taken back) change no bit."""
    from transformer_surgeon_b200 import ops
    lens = [1, 2, 3, 5, 7, 15, 16, 17, 30, 0]
    kv = make_kv(10, 4, 2, d, cuda, lens=lens)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(10, 64, 2, d, generator=g) for _ in range(2))
    q = torch.randn(10, 6, d, generator=g).to(DT[name]).to(cuda)
    zeros, outs = torch.zeros_like(kv.seq_lens), []
    for bad in (0.0, float("nan"), float("inf"), -float("inf")):
        for b, n in enumerate(lens):
            k[b, n:], v[b, n:] = bad, bad
        kv.append(k.to(cuda), v.to(cuda), seq_lens=zeros)
        outs.append(ops.paged_decode_attention(kv, q, 64))
    assert torch.isfinite(outs[0]).all()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])


def test_attention_passes_nan_on_where_it_counts(cuda):
    """A NaN among a head's cached values reaches that head's outputs and no other's."""
    from transformer_surgeon_b200 import ops
    kv = make_kv(2, 2, 2, 64, cuda, lens=[20, 20])
    x = torch.randn(2, 20, 2, 64, generator=torch.Generator().manual_seed(1)).to(cuda)
    bad = x.clone()
    bad[0, 3, 1, 5] = float("nan")
    kv.append(x, bad, seq_lens=torch.zeros_like(kv.seq_lens))
    out = ops.paged_decode_attention(kv, torch.ones(2, 4, 64, device=cuda), 32)
    assert torch.isnan(out[0, 2:, 5]).all() and torch.isnan(out).sum() == 2
    qn = torch.ones(2, 4, 64, device=cuda)
    qn[1, 0, 7] = float("nan")
    out = ops.paged_decode_attention(kv, qn, 32)
    assert torch.isnan(out[1, 0]).all() and not torch.isnan(out[1, 1:]).any()


@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_gather_and_prompt_attention(cuda, name):
    from transformer_surgeon_b200 import ops
    lens = [90, 90]
    kv = make_kv(2, 6, 2, 64, cuda, lens=lens)
    fill(kv, 90, 2)
    p, table = Plain(kv), kv.block_table.cpu().numpy()
    k, v = ops.kv_gather(kv, 90, dtype=DT[name])
    for got, x in ((k, p.k), (v, p.v)):
        want = x[table].transpose(0, 1, 3, 2, 4).reshape(2, 96, 2, 64)[:, :90]
        np.testing.assert_array_equal(got.double().cpu().numpy(), want)              # four significant bits: no rounding
    q = torch.randn(2, 37, 6, 64, generator=torch.Generator().manual_seed(3)).to(DT[name]).to(cuda)
    out = ops.prefill_attention(kv, q, 90).double().cpu().numpy()
    for i in (0, 17, 36):
        ref, size = plain_attention(kv, q[:, i], [90 - 37 + i + 1] * 2, 64 ** -0.5)
        assert (np.abs(out[:, i] - ref) <= 2 * tolerance(name, size, ref)).all()


# ------------------------------------------------------------------------------------------------ selection
def plain_select(logits, scores, n, finished=None, pad=0):
    """float64 on the CPU; the values of dead beams are -inf."""
    B, K = scores.shape
    x = logits.double().cpu().numpy().reshape(B, K, -1)
    s = scores.double().cpu().numpy()
    V = x.shape[-1]
    val = np.full((B, K, V), -np.inf)
    for b in range(B):
        for k in range(K):
            if not s[b, k] > -np.inf:
                continue
            if finished is not None and finished[b, k]:
                val[b, k, pad] = s[b, k]
                continue
            top = x[b, k].max()
            if np.isfinite(top):
                val[b, k] = s[b, k] + (x[b, k] - (top + np.log(np.exp(x[b, k] - top).sum())))
    flat = val.reshape(B, -1)
    at = np.argsort(-flat, axis=1, kind="stable")[:, :n]
    return np.take_along_axis(flat, at, 1), at // V + np.arange(B)[:, None] * K, at % V


def check_select(logits, scores, n, finished=None, pad=0, close=2e-7):
    """Equal tokens and parents, except that two candidates whose values are closer than `close` (relative; the row sums come from fp32
    exponentials of 2^-22) may change places."""
    from transformer_surgeon_b200 import ops
    ref = plain_select(logits, scores, n + 1 if n < logits.numel() // scores.shape[0] else n, finished, pad)
    fin = None if finished is None else finished
    out = [o.cpu().numpy() for o in ops.beam_select(logits, scores, n, finished=fin, pad_token=pad)]
    again = [o.cpu().numpy() for o in ops.beam_select(logits, scores, n, finished=fin, pad_token=pad)]
    for a, b in zip(out, again):
        np.testing.assert_array_equal(a, b)
    val = ref[0]
    np.testing.assert_allclose(out[0], val[:, :n], rtol=2e-7, atol=1e-6)
    for b in range(val.shape[0]):
        for i in range(n):
            if out[1][b, i] != ref[1][b, i] or out[2][b, i] != ref[2][b, i]:
                near = [j for j in range(max(0, i - 1), min(val.shape[1], i + 2)) if j != i and ref[1][b, j] != ref[1][b, i]]
                assert any(abs(val[b, j] - val[b, i]) <= close * abs(val[b, i]) for j in near), (b, i, out[1][b], ref[1][b], out[2][b], ref[2][b])
    return out


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 2, 7, 14), (3, 4, 33, 8), (2, 3, 1000, 6), (1, 4, 128256, 8), (2, 5, 50257, 32), (17, 2, 4097, 4),
                                     (1, 1, 8191, 32), (160, 2, 9001, 3), (1, 40, 2000, 32)])
def test_select(cuda, name, B, K, V, n):
    g = torch.Generator().manual_seed(V + n)
    logits = (torch.randn(B * K, V, generator=g) * 3).to(DT[name]).to(cuda)
    scores = (-5 * torch.rand(B, K, generator=g)).to(cuda)
    check_select(logits, scores, n)


@pytest.mark.parametrize("name", ["bf16", "fp32"])
@pytest.mark.parametrize("kind", ["one value", "few values", "ascending", "descending", "few allowed", "lowest", "none allowed", "peak late"])
def test_select_hard_rows(cuda, name, kind):
    """Ties, orders that move the bound all the time, masks."""
    B, K, V, n = 2, 3, 40000, 8
    g = torch.Generator().manual_seed(11)
    x = torch.randn(B * K, V, generator=g)
    if kind == "one value":
        x[:] = 1.5
    elif kind == "few values":
        x = torch.randint(0, 3, (B * K, V), generator=g).float()
    elif kind == "ascending":
        x = torch.linspace(-20, 20, V).expand(B * K, V).clone()
    elif kind == "descending":
        x = torch.linspace(20, -20, V).expand(B * K, V).clone()
    elif kind in ("few allowed", "none allowed", "lowest"):
        keep = torch.rand(B * K, V, generator=g) < (0.0001 if kind != "none allowed" else -1)
        x = torch.where(keep, x, torch.tensor(float("-inf") if kind != "lowest" else torch.finfo(DT[name]).min))
    else:
        x[:, -3:] += 200
    logits = x.to(DT[name]).to(cuda)
    scores = torch.tensor([[-1.0, -1.0, -2.5], [0.0, -3.0, -0.25]], device=cuda)     # rows of equal scores: ties across beams
    check_select(logits, scores, n)


def test_select_more_sequences_than_counters(cuda):
    g = torch.Generator().manual_seed(2)
    logits, scores = torch.randn(2 * 4100, 40, generator=g).to(cuda), -torch.rand(4100, 2, generator=g).to(cuda)
    check_select(logits, scores, 3)


def test_select_dead_and_finished_beams(cuda):
    B, K, V, n = 6, 4, 5000, 8
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(B * K, V, generator=g).to(cuda)
    scores = -torch.rand(B, K, generator=g).to(cuda)
    scores[0, 1:] = float("-inf")                                # a search's first step
    scores[1] = float("-inf")
    scores[2, 0] = float("nan")
    logits[3 * K + 1, 77], logits[3 * K + 2, 5] = float("nan"), float("inf")
    finished = torch.zeros(B, K, dtype=torch.bool, device=cuda)
    finished[4, :] = True
    finished[5, 2] = True
    scores[5, 2] = 3.0
    finished[0, 2] = True                                        # finished, and dead
    v, p, t = check_select(logits, scores, n, finished, pad=3)
    assert t[5, 0] == 3 and p[5, 0] == 5 * K + 2 and v[5, 0] == 3.0
    assert sorted(p[4, :4]) == [16, 17, 18, 19] and (t[4, :4] == 3).all() and (v[4, 4:] == -np.inf).all()
    assert list(t[4, 4:]) == [0, 1, 2, 4] and (p[4, 4:] == 16).all() and list(t[1]) == list(range(n))


@pytest.mark.parametrize("name,stride,start", [("bf16", 1003, 1), ("bf16", 1024, 8), ("fp32", 1001, 3), ("fp32", 1004, 2)])
def test_select_strided_rows(cuda, name, stride, start):
    g = torch.Generator().manual_seed(4)
    buf = torch.full((6 * stride + 16,), float("nan")).to(DT[name]).to(cuda)         # a read outside of the rows shows
    rows = buf[start:start + 6 * stride].view(6, stride)[:, :1000]
    rows.copy_(torch.randn(6, 1000, generator=g))
    check_select(rows, -torch.rand(2, 3, generator=g).to(cuda), 6)
    check_select(rows.unflatten(0, (2, 3)).flatten(0, 1), -torch.rand(2, 3, generator=g).to(cuda), 6)


# ------------------------------------------------------------------------------------------------ reordering
def kvs_of(fmt, layers, R, pages, hkv, d, dev):
    from transformer_surgeon_b200 import ops
    table = torch.randperm(R * pages + 3, generator=torch.Generator().manual_seed(2))[:R * pages].to(torch.int32).reshape(R, pages).to(dev)
    lens = torch.zeros(R, dtype=torch.int32, device=dev)
    kvs = [ops.PagedKV(fmt, R * pages + 3, hkv, d, table, lens, dev) for _ in range(layers)]
    g = torch.Generator().manual_seed(3)
    for kv in kvs:
        for p in (kv.k_pool, kv.v_pool):
            p.copy_(torch.randint(0, 256, p.shape, generator=g, dtype=torch.uint8))
        if kv.k_scale is not None:
            kv.k_scale.copy_(torch.rand(R, hkv, generator=g))
            kv.v_scale.copy_(torch.rand(R, hkv, generator=g))
    return kvs


@pytest.mark.parametrize("fmt", ["fp8_page", "fp8", "int8", "nvfp4", "bf16", "fp32"])
@pytest.mark.parametrize("R,pages,layers", [(4, 5, 3), (33, 3, 1), (300, 2, 1), (1, 4, 2)])
def test_reorder(cuda, fmt, R, pages, layers):
    """Tables, pages and scales after several reorderings, parents named twice, out of range, of other lengths, and permutations among them."""
    from transformer_surgeon_b200 import ops
    kvs = kvs_of(fmt, layers, R, pages, 3, 64, cuda)
    a = kvs[0]
    reorder = ops.BeamReorder(kvs)
    home = a.block_table.cpu().numpy().copy()
    table = home.copy()
    pools = [p.cpu().numpy().copy() for kv in kvs for p in (kv.k_pool, kv.v_pool)]
    scales = [p.cpu().numpy().copy() for kv in kvs for p in (kv.k_scale, kv.v_scale) if p is not None]
    g = np.random.default_rng(R)
    for step, length in enumerate([16 * pages, 1, 16, 17, 16 * pages - 1]):
        lens = np.full(R, length, dtype=np.int32)
        if step == 3:
            lens[R // 2:] += 1                                   # two groups of other lengths
        parents = g.permutation(R) if step == 1 else g.integers(0, R, R)
        if R > 3:
            parents[1], parents[2] = (-1, R) if step != 1 else (parents[1], parents[2])
        if step == 1:                                            # shorter than before: sequences started anew, with pages of their own
            reorder.reset()
            table = home.copy()
        a.seq_lens.copy_(torch.from_numpy(lens))
        reorder(torch.from_numpy(parents.astype(np.int32)).to(cuda))
        moved = [(r, p) for r, p in enumerate(parents) if 0 <= p < R and lens[p] == lens[r]]
        old, old_pools, old_scales = table.copy(), [p.copy() for p in pools], [s.copy() for s in scales]
        for r, p in moved:
            full = lens[r] // PAGE
            table[r, :full] = old[p, :full]
            if lens[r] % PAGE:
                for x, y in zip(pools, old_pools):
                    x[home[r, full]] = y[home[p, full]]
            for x, y in zip(scales, old_scales):
                x[r] = y[p]
        np.testing.assert_array_equal(a.block_table.cpu().numpy(), table)
        for x, p in zip(pools, [p for kv in kvs for p in (kv.k_pool, kv.v_pool)]):
            np.testing.assert_array_equal(p.cpu().numpy(), x)
        for x, p in zip(scales, [p for kv in kvs for p in (kv.k_scale, kv.v_scale)]):
            np.testing.assert_array_equal(p.cpu().numpy(), x)
    a.seq_lens.zero_()
    reorder(torch.zeros(R, dtype=torch.int32, device=cuda))      # nothing cached: nothing moves
    np.testing.assert_array_equal(a.block_table.cpu().numpy(), table)
    reorder.reset()
    np.testing.assert_array_equal(a.block_table.cpu().numpy(), home)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("name", ["bf16", "fp32"])
def test_beams_of_one_layer_follow_their_histories(cuda, name):
    """append, select and reorder over 40 steps: every beam's attention is that of a cache that holds its own history alone."""
    from transformer_surgeon_b200 import ops
    B, K, hkv, g, d, T, V = 2, 3, 2, 4, 64, 21, 300
    R = B * K
    kv = make_kv(R, 5, hkv, d, cuda)
    reorder = ops.BeamReorder([kv])
    gen = torch.Generator().manual_seed(1)
    prompt = torch.randn(2, B, T, hkv, d, generator=gen).to(DT[name]).to(cuda).repeat_interleave(K, dim=1)
    kv.append(prompt[0], prompt[1])
    kv.seq_lens += T
    history = [prompt[:, r].clone() for r in range(R)]            # per beam: [2, tokens, hkv, d]
    scores = torch.zeros(B, K, device=cuda)
    for step in range(40):
        logits = torch.randn(R, V, generator=gen).to(cuda)
        scores, parents, tokens = ops.beam_select(logits, scores, K)
        reorder(parents.view(-1))
        history = [history[p] for p in parents.view(-1).tolist()]
        new = torch.randn(2, R, 1, hkv, d, generator=gen).to(DT[name]).to(cuda)
        kv.append(new[0], new[1])
        kv.seq_lens += 1
        history = [torch.cat((h, new[:, r]), 1) for r, h in enumerate(history)]
        if step in (0, 10, 11, 26, 39):
            alone = make_kv(R, 5, hkv, d, cuda, seed=7)
            for t0, t1 in [(0, T)] + [(t, t + 1) for t in range(T, T + step + 1)]:
                x = torch.stack([h[:, t0:t1] for h in history], 1)
                alone.append(x[0], x[1], seq_lens=torch.full((R,), t0, dtype=torch.int32, device=cuda))
            alone.seq_lens += T + step + 1
            q = torch.randn(R, hkv * g, d, generator=gen).to(DT[name]).to(cuda)
            assert torch.equal(ops.paged_decode_attention(kv, q, 80), ops.paged_decode_attention(alone, q, 80))


def tiny_engine(cuda, batch, kv_format, dtype=torch.float32):
    from tests.test_gpu_hf import tiny
    from transformer_surgeon_b200 import surgeon
    model = tiny("llama", torch.float32)
    return model, surgeon.decoder_from_model(model.to(dtype), batch, 64, kv_format)


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("kv_format", ["fp32", "fp8_page", "fp8", "int8"])
def test_engine_beam_search(cuda, captured, kv_format):
    """CompressedDecoder.beam_search against a search that feeds every beam's whole sequence to a fresh cache each step."""
    B, K, T, new = 2, 3, 9, 12
    model, dec = tiny_engine(cuda, B * K, kv_format)
    if captured:
        dec.capture()
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(5)).cuda()
    seqs, scores = dec.beam_search(ids, new, K)
    twice, _ = dec.beam_search(ids, new, K)                       # pages are the rows' own again
    assert torch.equal(seqs, twice) and torch.equal(seqs[:, :, :T], ids[:, None].expand(B, K, T))
    _, ref = tiny_engine(cuda, B * K, kv_format)
    rows, total = ids.repeat_interleave(K, 0), torch.full((B, K), float("-inf"), dtype=torch.float64, device=cuda)
    total[:, 0] = 0
    for i in range(new):
        ref.prefill(rows[:, :T])
        for t in range(T, rows.shape[1]):
            ref.step(rows[:, t])
        value = (total[..., None] + torch.log_softmax(ref.logits.double(), -1).view(B, K, -1)).flatten(1)
        total, at = value.topk(K)
        rows = torch.cat((rows.view(B, K, -1).gather(1, (at // 512)[..., None].expand(B, K, rows.shape[1])), (at % 512)[..., None]), 2).flatten(0, 1)
    assert torch.equal(rows.view(B, K, -1), seqs)
    assert torch.allclose(total.float(), scores, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("kv_format,dtype", [("fp8_page", torch.bfloat16), ("nvfp4", torch.bfloat16), ("fp8", torch.float32)])
@pytest.mark.parametrize("T", [1, 16, 37])
def test_prompt_once_for_all_beams(cuda, kv_format, dtype, T):
    """The rows of a prompt hold what each holds that went through the model by itself, up to the order of sums in layers of other token counts."""
    _, a = tiny_engine(cuda, 6, kv_format, dtype)
    _, b = tiny_engine(cuda, 6, kv_format, dtype)
    ids = torch.randint(0, 512, (2, T), generator=torch.Generator().manual_seed(5)).cuda()
    one, each = a.prefill(ids, beams=3).clone(), b.prefill(ids.repeat_interleave(3, 0)).clone()
    tol = 2e-2 if dtype == torch.bfloat16 else 2e-3
    for _ in range(3):
        assert (one - each).abs().max() <= tol * each.abs().max()
        tokens = each.argmax(-1)
        one, each = a.step(tokens).clone(), b.step(tokens).clone()
    assert torch.equal(a.seq_lens, b.seq_lens)


def test_engine_beam_search_ends(cuda):
    """A beam that has met the end token is padded and keeps its score; greedy decoding afterwards is what it was before."""
    _, dec = tiny_engine(cuda, 4, "fp8_page")
    ids = torch.randint(0, 512, (1, 9), generator=torch.Generator().manual_seed(5)).cuda()
    greedy, _ = dec.generate(ids.expand(4, 9), 10, batched_prefill=True)
    free, _ = dec.beam_search(ids, 10, 4)
    end = int(free[0, 0, 12])                                     # a token that the best beam meets early
    seqs, scores = dec.beam_search(ids, 10, 4, eos_token_id=end, pad_token_id=0)
    for s in seqs[0, :, 9:].tolist():
        if end in s:
            assert all(t == 0 for t in s[s.index(end) + 1:])
    assert (scores[0, 1:] <= scores[0, :-1]).all()
    assert torch.equal(dec.generate(ids.expand(4, 9), 10, batched_prefill=True)[0], greedy)
    with pytest.raises(ValueError):
        dec.beam_search(ids, 10, 3)
    with pytest.raises(ValueError):
        dec.beam_search(ids, 60, 4)


def test_blocks_path_with_pages_of_their_own_scales(cuda):
    """The engine token by token against the prompt in one pass: no scales to set beforehand.  Logits a few e4m3 roundings (2^-4 of a value) apart,
    as the pages' scales grow in other steps; within 2 % of the largest."""
    _, a = tiny_engine(cuda, 2, "fp8_page")
    _, b = tiny_engine(cuda, 2, "fp8_page")
    ids = torch.randint(0, 512, (2, 21), generator=torch.Generator().manual_seed(5)).cuda()
    one = a.prefill(ids).clone()
    b.reset()
    for t in range(21):
        stepwise = b.step(ids[:, t])
    assert (one - stepwise).abs().max() <= 2e-2 * one.abs().max()
    assert torch.equal(a.seq_lens, b.seq_lens)


@pytest.mark.parametrize("fmt", ["fp32", "fp8_page"])
def test_hf_beam_search(cuda, fmt):
    """generate(num_beams=...) of Hugging Face over the paged cache: fp32 pages give the stock cache's sequences."""
    from tests.test_gpu_hf import tiny
    from transformer_surgeon_b200 import hf_cache
    model = tiny("qwen2", torch.float32)
    ids = torch.randint(0, 512, (2, 19), generator=torch.Generator().manual_seed(5)).cuda()
    args = dict(attention_mask=torch.ones_like(ids), max_new_tokens=30, min_new_tokens=30, do_sample=False, num_beams=3, pad_token_id=0, eos_token_id=None)
    stock = model.generate(ids, **args)
    model.config._attn_implementation = hf_cache.ATTN_NAME
    cache = hf_cache.PagedQuantCache(model.config, batch=6, max_len=64, kv_format=fmt)
    out = model.generate(ids, past_key_values=cache, **args)
    assert out.shape == stock.shape
    if fmt == "fp32":
        assert torch.equal(out, stock)
    cache.reset()
    assert torch.equal(model.generate(ids, past_key_values=cache, **args), out)


def test_select_and_reorder_captured(cuda):
    """One CUDA graph of selection, reordering, append and attention, replayed on other inputs and beside an eager call on another stream."""
    from transformer_surgeon_b200 import ops
    R, hkv, d, V = 4, 1, 64, 1000
    kv = make_kv(R, 4, hkv, d, cuda, lens=[20] * R)
    fill(kv, 20, 1)
    reorder = ops.BeamReorder([kv])
    state = kv.k_pool.clone(), kv.v_pool.clone(), kv.block_table.clone()
    logits, scores = torch.zeros(R, V, device=cuda), torch.zeros(1, R, device=cuda)
    k, v, q = (torch.zeros(R, 1, h, d, device=cuda) for h in (hkv, hkv, 2))

    def put(seed):
        g = torch.Generator().manual_seed(seed)
        for t in (logits, scores, k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        kv.k_pool.copy_(state[0]), kv.v_pool.copy_(state[1]), kv.block_table.copy_(state[2])

    def run(ws_s, ws_a):
        out = ops.beam_select(logits, scores, R, ws=ws_s)
        reorder(out[1].view(-1))
        kv.append(k, v)
        return (*out, ops.paged_decode_attention(kv, q[:, 0], 64, ws=ws_a, seq_lens=kv.seq_lens + 1))
    size = ops.beam_select_workspace_bytes(1, R, V, torch.float32, R), ops.decode_attn_workspace_bytes(R, 2, d, 64)
    new_ws = lambda: [torch.zeros(n, dtype=torch.uint8, device=cuda) for n in size]  # noqa: E731
    put(1)
    run(*new_ws())
    side = torch.cuda.Stream()
    graph, ws = torch.cuda.CUDAGraph(), new_ws()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = run(*ws)
    for seed in (2, 3):
        put(seed)
        want = [x.clone() for x in run(*new_ws())]
        put(seed)
        other = torch.randn(3 * R, 777, device=cuda)
        side.wait_stream(torch.cuda.current_stream())
        graph.replay()
        with torch.cuda.stream(side):
            beside = ops.beam_select(other, torch.zeros(3, R, device=cuda), 2, ws=new_ws()[0].new_zeros(1 << 20))
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        assert torch.equal(beside[2], ops.beam_select(other, torch.zeros(3, R, device=cuda), 2)[2])


def test_default_scratch_is_of_one_stream_and_of_one_graph(cuda):
    """Selection and attention without a workspace: on two streams at once, in two graphs replayed at once, and eagerly after a capture that never ran."""
    from transformer_surgeon_b200 import ops
    jobs = []
    for i, (B, K, V) in enumerate(((5, 4, 70001), (2, 7, 90002))):
        kv = make_kv(B * K, 40, 1, 64, cuda, seed=i, lens=[600 - 17 * r for r in range(B * K)])
        fill(kv, 600, i)
        g = torch.Generator().manual_seed(i)
        args = torch.randn(B * K, V, generator=g).to(cuda), torch.randn(B, K, generator=g).to(cuda), kv, torch.randn(B * K, 8, 64, generator=g).to(cuda)
        ws = [torch.zeros(n, dtype=torch.uint8, device=cuda)
              for n in (ops.beam_select_workspace_bytes(B, K, V, torch.float32, K), ops.decode_attn_workspace_bytes(B * K, 8, 64, 640))]

        def run(args=args, ws=(None, None)):
            logits, scores, kv, q = args
            return (*ops.beam_select(logits, scores, ws=ws[0]), ops.paged_decode_attention(kv, q, 640, ws=ws[1]))
        jobs.append((run, [x.clone() for x in run(ws=ws)], torch.cuda.Stream()))

    def at_once(calls):
        torch.cuda.synchronize()
        outs = []
        for call, (_, _, stream) in zip(calls, jobs):
            with torch.cuda.stream(stream):
                for _ in range(4):
                    out = call()
                outs.append(out)
        torch.cuda.synchronize()
        for out, job in zip(outs, jobs):
            for a, b in zip(out, job[1]):
                assert torch.equal(a, b)
    graphs, outs = [], []
    for run, _, _ in jobs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run())
    at_once([run for run, _, _ in jobs])
    at_once([lambda graph=graph, out=out: (graph.replay(), out)[1] for graph, out in zip(graphs, outs)])
    at_once([run for run, _, _ in jobs])


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(cuda):
    from transformer_surgeon_b200 import ops
    logits, scores = torch.zeros(4, 50, device=cuda), torch.zeros(2, 2, device=cuda)
    for args, kw in (((logits, scores, 33), {}), ((logits, scores, 0), {}), ((logits[:, :3], scores, 7), {}),
                     ((logits, scores, 2), dict(finished=torch.zeros(2, 2, dtype=torch.bool, device=cuda), pad_token=50)),
                     ((logits, scores, 2), dict(ws=torch.zeros(64, dtype=torch.uint8, device=cuda)))):
        with pytest.raises(ops.Tsb200Error):
            ops.beam_select(*args, **kw)
    kv = make_kv(2, 2, 1, 64, cuda)
    k = torch.zeros(2, 1, 1, 64, device=cuda)
    cos, sin = rope_tables(64, 8, cuda)
    with pytest.raises(ops.Tsb200Error):
        kv.append(k, k, rope=(cos.view(-1)[1:].view(-1)[:32 * 7].view(7, 32), sin[:7]))       # tables off their 16 bytes
    with pytest.raises(ops.Tsb200Error):
        ops.paged_decode_attention(kv, torch.zeros(2, 1, 64, device=cuda), 33)                  # beyond the block table
    with pytest.raises(ops.Tsb200Error):
        ops.PagedKV("fp8_page", 2, 1, 96, kv.block_table, kv.seq_lens, cuda).append(torch.zeros(2, 1, 1, 96, device=cuda), torch.zeros(2, 1, 1, 96, device=cuda))
    with pytest.raises(ValueError):
        ops.PagedKV("fp8_page", 4, 1, 64, kv.block_table, kv.seq_lens, cuda, k_pool=torch.zeros(4, 1, 1024, dtype=torch.uint8, device=cuda))
    other = make_kv(2, 2, 1, 64, cuda)
    with pytest.raises(ValueError):
        ops.BeamReorder([kv, other])                              # another block table
    many = make_kv(2049, 1, 1, 64, cuda)
    with pytest.raises(ops.Tsb200Error):
        ops.BeamReorder([many])(torch.zeros(2049, dtype=torch.int32, device=cuda))           # more rows than a CTA takes
    kv.block_table[1] = kv.block_table[0]
    with pytest.raises(ValueError):
        ops.BeamReorder([kv])                                     # rows without pages of their own
    with pytest.raises(ValueError):
        ops.BeamReorder([other])(torch.zeros(2, dtype=torch.int64, device=cuda))


@pytest.mark.parametrize("fmt", ["fp8_page", "int8"])
def test_refusals_of_shared_memory_and_of_other_shapes(cuda, fmt):
    """Expanded tensors (a stride of 0, which the C entries take for "dense"), tensors of another type or shape, more sequences than the cache has."""
    from transformer_surgeon_b200 import ops
    for logits, scores in ((torch.zeros(1, 50, device=cuda).expand(4, 50), torch.zeros(2, 2, device=cuda)),
                           (torch.zeros(1, 1, 50, device=cuda).expand(2, 2, 50), torch.zeros(2, 2, device=cuda))):
        with pytest.raises(ValueError, match="share memory"):
            ops.beam_select(logits, scores)
    table = torch.arange(6, dtype=torch.int32, device=cuda).reshape(3, 2)
    kv = ops.PagedKV(fmt, 6, 2, 64, table, torch.full((3,), 5, dtype=torch.int32, device=cuda), cuda)
    rope = rope_tables(64, 32, cuda)
    x = torch.zeros(3, 2, 2, 64, device=cuda)
    for bad in (x[:1].expand(3, 2, 2, 64)[:, :1], x[:, :1].expand(3, 2, 2, 64), x[:1, :1].expand(3, 2, 2, 64)):
        for call in (lambda: kv.append(bad, bad), lambda: kv.rope_append(bad, x[:, :bad.shape[1]], x[:, :bad.shape[1]], rope)):
            with pytest.raises(ValueError):
                call()
    for call in (lambda: kv.append(x, x.bfloat16()), lambda: kv.append(x, x[:, :1]), lambda: kv.append(x[:, :, :1], x[:, :, :1]),
                 lambda: kv.append(x.repeat(2, 1, 1, 1), x.repeat(2, 1, 1, 1)), lambda: kv.append(x, x, seq_lens=kv.seq_lens[:2]),
                 lambda: kv.rope_append(x.bfloat16(), x, x, rope), lambda: kv.rope_append(x[:2], x, x, rope),
                 lambda: ops.paged_decode_attention(kv, x[:1, 0].expand(3, 2, 64), 32), lambda: ops.paged_decode_attention(kv, x.view(6, 2, 64), 32),
                 lambda: ops.paged_decode_attention(kv, x.view(3, 2, 128), 32)):
        with pytest.raises(ValueError):
            call()
    ops.paged_decode_attention(kv, x[:, 0], 32)
    torch.cuda.synchronize()


def test_prompt_of_32_bits_with_overlapping_launches(cuda):
    """The attention of a prompt chunk behind the append that wrote its pages, the engine's way (lengths and tables made once for all layers)."""
    from transformer_surgeon_b200 import ops
    outs = []
    for pdl in (False, True):
        kv = make_kv(2, 40, 2, 64, cuda, lens=[600, 600])
        x = torch.randn(3, 2, 600, 2, 64, generator=torch.Generator().manual_seed(5)).to(cuda)
        sequences, zeros = ops.query_sequences(kv, 2, 600, 600), torch.zeros_like(kv.seq_lens)
        torch.cuda.synchronize()
        old = ops.set_pdl(pdl)
        try:
            kv.append(x[1], x[2], seq_lens=zeros)
            outs.append(ops.prefill_attention(kv, x[0].contiguous(), 600, sequences=sequences))
            torch.cuda.synchronize()
        finally:
            ops.set_pdl(old)
    assert torch.equal(outs[0], outs[1])
