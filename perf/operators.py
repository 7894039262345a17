"""Beam search over an 8-bit paged cache whose pages carry their own scales: the operators, in plain form and as the framework's calls.

  append    keys and values of new tokens into pages of 16 tokens, the rotation of keys and queries on the way (ops.PagedKV.rope_append,
            format "fp8_page": e4m3 codes, one power-of-two scale per page and head)
  attention one query token per sequence over such pages (ops.paged_decode_attention)
  select    the n best continuations over beams and vocabulary (ops.beam_select)
  reorder   the cached tokens of every layer follow the beams that were selected (ops.BeamReorder)

Head layouts, vocabularies and layer counts are those of Llama-3-8B, Qwen2.5-VL-7B and Qwen2-0.5B, which the repository's configurations
use.  Cached values are N(0, 1) with four outlier channels a head (x 20); logits are N(0, 2.5^2).

A page record of a kv head is 16 * d code bytes (K: [token][element], V: [element][token]) and 16 bytes whose first four are the fp32 scale.
"""
import math

import torch

own = False

HEADS = {"llama3-8b": (32, 8, 128), "qwen2.5-vl-7b": (28, 4, 128), "qwen2-0.5b": (14, 2, 64)}      # query heads, kv heads, head size
VOCAB = {"llama3-8b": 128256, "qwen2.5-vl-7b": 152064, "qwen2-0.5b": 151936}
PAGE = 16
EXP_LO, EXP_HI = -40, 40                    # exponents a page's scale may have
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a decode step of many beams
        dict(name="append_b64", op="append", arch="llama3-8b", batch=64, tokens=1, context=2048, dtype="bf16"),
        # an odd chunk behind a cached prompt, an fp32 model
        dict(name="append_chunk77", op="append", arch="qwen2-0.5b", batch=3, tokens=77, context=301, dtype="fp32"),
        # the prompts of a batch
        dict(name="append_prompt", op="append", arch="llama3-8b", batch=16, tokens=2048, context=0, dtype="bf16"),
        # four beams of one stream, a short context
        dict(name="attn_b4", op="attention", arch="qwen2-0.5b", batch=4, context=519, dtype="fp32"),
        # a decode batch at the benchmark's context
        dict(name="attn_b32", op="attention", arch="llama3-8b", batch=32, context=2100, dtype="bf16"),
        # few beams over a long document, seven query heads to a kv head
        dict(name="attn_b8_32k", op="attention", arch="qwen2.5-vl-7b", batch=8, context=32768, dtype="bf16"),
        # a large serving batch
        dict(name="attn_b64_8k", op="attention", arch="llama3-8b", batch=64, context=8192, dtype="bf16"),
        # four beams of one sequence
        dict(name="select_b1", op="select", arch="llama3-8b", batch=1, beams=4, best=8, vocab=128256, dtype="bf16", finished=False),
        # fp32 logits, an odd number of beams, some of them finished
        dict(name="select_b5_fp32", op="select", arch="qwen2-0.5b", batch=5, beams=3, best=6, vocab=151936, dtype="fp32", finished=True),
        # a batch of beam searches over the widest vocabulary
        dict(name="select_b32", op="select", arch="qwen2.5-vl-7b", batch=32, beams=8, best=16, vocab=152064, dtype="bf16", finished=False),
        # four beams of one sequence, every layer's cache
        dict(name="reorder_b4", op="reorder", arch="qwen2-0.5b", batch=1, beams=4, layers=24, context=519),
        # sixteen sequences of four beams
        dict(name="reorder_b64", op="reorder", arch="llama3-8b", batch=16, beams=4, layers=32, context=333),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "select", "select", "reorder"])
    arch = rng.choice(sorted(HEADS))
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "append":
        batch = _log(rng, 1, 96)
        tokens = rng.choice([1, _log(rng, 1, 32768 // batch)])
        return dict(op=op, arch=arch, batch=batch, tokens=min(tokens, 4096), context=rng.randint(0, 1500), dtype=dtype)
    if op == "attention":
        batch = _log(rng, 1, 96)
        return dict(op=op, arch=arch, batch=batch, context=_log(rng, 17, min(32768, 400000 // batch)), dtype=dtype)
    if op == "select":
        beams = rng.randint(1, 12)
        vocab = rng.choice([VOCAB[arch], _log(rng, 1000, 152064), _log(rng, 1000, 152064)])
        batch = _log(rng, 1, max(1, min(64, 30000000 // (beams * vocab))))
        return dict(op=op, arch=arch, batch=batch, beams=beams, best=rng.choice([beams, 2 * beams, rng.randint(1, 32)]), vocab=vocab, dtype=dtype,
                    finished=rng.random() < 0.3)
    beams, layers = rng.randint(2, 8), rng.randint(2, 32)
    batch = _log(rng, 1, 64 // beams)
    per_token = layers * 2 * HEADS[arch][1] * (HEADS[arch][2] + 1)
    return dict(op=op, arch=arch, batch=batch, beams=beams, layers=layers, context=_log(rng, 17, max(18, min(4096, 400000000 // (per_token * batch * beams)))))


def work(case):
    H, hkv, d = HEADS[case["arch"]]
    size = 4 if case.get("dtype") == "fp32" else 2
    B = case["batch"]
    if case["op"] == "append":
        n = B * case["tokens"]
        return dict(bytes=n * (2 * H + 2 * hkv) * d * size + n * d * 4 + 2 * n * hkv * d, flops=n * (H + 2 * hkv) * d * 3)
    if case["op"] == "attention":
        n = int(_lengths(case).sum())
        return dict(bytes=n * 2 * hkv * (d + 1) + B * 2 * H * d * size, flops=4 * n * H * d)
    if case["op"] == "select":
        n = B * case["beams"] * case["vocab"]
        return dict(bytes=n * size + B * case["best"] * 16, flops=4 * n)
    rows, open_tokens = B * case["beams"], case["context"] % PAGE
    table = rows * (case["context"] // PAGE) * 4 * 2
    return dict(bytes=table + 2 * rows * 3 // 4 * case["layers"] * 2 * hkv * d * open_tokens, flops=0)


def _lengths(case):
    """Tokens cached per sequence: unequal, the longest at the context."""
    B, L = case["batch"], case["context"]
    at = torch.arange(B, dtype=torch.int64)
    lens = L - (at * 977 % max(1, L // 2 + 1))
    return lens if case["op"] != "append" or case["context"] else torch.zeros_like(lens)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    H, hkv, d = HEADS[case["arch"]]
    dt, B = TYPES[case.get("dtype", "bf16")], case["batch"]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "select":
        K = case["beams"]
        logits = (normal(B * K, case["vocab"]) * 2.5).to(dt)
        scores = -normal(B, K).abs() * 2 - 5
        finished = (torch.rand(B, K, generator=g, device="cuda") < 0.3) if case["finished"] else None
        return dict(case=case, logits=logits, scores=scores, finished=finished)
    if case["op"] == "reorder":
        K = case["beams"]
        R = B * K
        pages = (case["context"] + 64 + PAGE - 1) // PAGE
        pool = torch.randint(0, 256, (case["layers"], 2, R * pages, hkv, PAGE * d + 16), generator=g, device="cuda", dtype=torch.uint8)
        table = torch.arange(R * pages, dtype=torch.int32, device="cuda").reshape(R, pages)
        lens = torch.full((R,), case["context"], dtype=torch.int32, device="cuda")
        parents = (torch.randint(0, K, (B, K), generator=g, device="cuda") + K * torch.arange(B, device="cuda")[:, None]).reshape(-1).to(torch.int32)
        state = dict(case=case, pool=pool, table=table, lens=lens, parents=parents)
        if own:
            state["kvs"] = [_own_kv(pool[i], table, lens, hkv, d) for i in range(case["layers"])]
            state["reorder"] = _ops().BeamReorder(state["kvs"])
        return state
    lens = _lengths(case)
    new = case.get("tokens", 0)
    pages = (int(lens.max()) + new + PAGE - 1) // PAGE
    table = torch.randperm(B * pages, generator=g, device="cuda").to(torch.int32).reshape(B, pages)
    pool = torch.zeros((2, B * pages, hkv, PAGE * d + 16), dtype=torch.uint8, device="cuda")
    # cached codes: N(0, 64^2) at scales around 2^-6, outlier channels at the end of the range
    spread = torch.full((d,), 22.0, device="cuda")
    spread[:: d // 4] = 440.0
    scales = torch.pow(2.0, torch.randint(-7, -3, (2, B * pages, hkv), generator=g, device="cuda").float())
    if case["op"] == "attention" or case["context"]:
        for side in range(2):
            for at in range(0, B * pages, 4096):
                n = min(4096, B * pages - at)
                codes = (normal(n, hkv, PAGE, d) * spread).clamp(-448, 448).to(torch.float8_e4m3fn)
                codes = codes if side == 0 else codes.transpose(2, 3).contiguous()
                pool[side, at:at + n, :, :PAGE * d] = codes.view(torch.uint8).reshape(n, hkv, PAGE * d)
        pool.view(torch.float32)[..., PAGE * d // 4] = scales
    lens = lens.to(device="cuda", dtype=torch.int32)
    state = dict(case=case, pool=pool, table=table, lens=lens)
    if own:
        state["kv"] = _own_kv(pool, table, lens, hkv, d)
    if case["op"] == "attention":
        state["q"] = normal(B, H, d).to(dt)
        return state
    # q, k and v as a projection leaves them: column slices of one [tokens, (H + 2 hkv) d] matrix; keys and values with outlier channels
    x = normal(B, new, H + 2 * hkv, d)
    x[:, :, H:, :: d // 4] *= 20
    x = x.to(dt).reshape(B * new, (H + 2 * hkv) * d)
    state["q"], state["k"], state["v"] = (
        x[:, a * d:b * d].unflatten(1, (b - a, d)).unflatten(0, (B, new)) for a, b in ((0, H), (H, H + hkv), (H + hkv, H + 2 * hkv)))
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device="cuda").double() / d))
    angle = torch.arange(pages * PAGE, device="cuda").double()[:, None] * inv
    state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    return state


def _ops():
    from transformer_surgeon_b200 import ops
    return ops


def _own_kv(pool, table, lens, hkv, d):
    return _ops().PagedKV("fp8_page", pool.shape[1], hkv, d, table, lens, pool.device, k_pool=pool[0], v_pool=pool[1])


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if op == "append":
        return _append(state)
    if op == "attention":
        return _attention(state)
    if op == "select":
        return _select(state)
    return _reorder(state)


def _append(state):
    pool, d = state["pool"], state["q"].shape[-1]
    if own:
        state["kv"].rope_append(state["q"], state["k"], state["v"], (state["cos"], state["sin"]))
    else:
        q, k, v, lens = state["q"], state["k"].float(), state["v"].float(), state["lens"].long()
        B, T = q.shape[:2]
        at = lens[:, None] + torch.arange(T, device=q.device)
        cos, sin = state["cos"][at][:, :, None], state["sin"][at][:, :, None]
        k = _rotated(k, cos, sin)
        q.copy_(_rotated(q.float(), cos, sin))
        # the pages that get tokens; a page number past a sequence's last one stands for the last one once more
        touched = (lens % PAGE + T + PAGE - 1) // PAGE
        nth = torch.minimum(torch.arange((T + 2 * PAGE - 2) // PAGE, device=q.device)[None], touched[:, None] - 1)
        ids = state["table"].long().gather(1, lens[:, None] // PAGE + nth)
        slot = (nth * PAGE)[:, :, None] + torch.arange(PAGE, device=q.device)         # [B, pages, 16]: slot counted from the first page's start
        j = slot - (lens % PAGE)[:, None, None]
        is_new, is_old = (j >= 0) & (j < T), j < 0
        for side, x in ((0, k), (1, v)):
            x = x[torch.arange(B, device=q.device)[:, None, None], j.clamp(0, T - 1)]  # [B, pages, 16, hkv, d]
            x = x.masked_fill(~is_new[..., None, None], 0.0).transpose(2, 3)           # [B, pages, hkv, 16, d]
            codes = pool[side, :, :, :PAGE * d]
            scale = pool[side].view(torch.float32)[:, :, PAGE * d // 4]
            old = codes[ids].view(torch.float8_e4m3fn).float()
            old = old.unflatten(3, (PAGE, d)) if side == 0 else old.unflatten(3, (d, PAGE)).transpose(3, 4)
            amax = x.abs().masked_fill(~x.isfinite(), 0.0).amax((3, 4))
            m, e = torch.frexp(amax)                                                   # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
            s = torch.pow(2.0, torch.where(amax > 0, e - 9 + (m > 0.875).int(), EXP_LO).clamp(EXP_LO, EXP_HI).float())
            had = is_old.any(2)[..., None]
            s = torch.where(had, torch.maximum(s, scale[ids]), s)
            y = torch.where(is_new[:, :, None, :, None], x / s[..., None, None], old * (scale[ids] / s)[..., None, None])
            y = y.masked_fill(~(is_new | is_old)[:, :, None, :, None], 0.0).clamp(-448, 448).to(torch.float8_e4m3fn)
            y = y if side == 0 else y.transpose(3, 4)
            codes[ids] = y.reshape(*ids.shape, -1, PAGE * d).view(torch.uint8)
            scale[ids] = s
    out = {"q": state["q"]}
    for side, name in ((0, "k"), (1, "v")):
        out[name] = pool[side, :, :, :PAGE * d].view(torch.float8_e4m3fn)
        out[name + "_scale"] = pool[side].view(torch.float32)[:, :, PAGE * d // 4]
    return out


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _attention(state):
    q, lens = state["q"], state["lens"]
    B, H, d = q.shape
    if own:
        return _ops().paged_decode_attention(state["kv"], q, state["case"]["context"])
    pool, table = state["pool"], state["table"].long()
    hkv, L = pool.shape[2], table.shape[1] * PAGE
    codes = pool[..., :PAGE * d].view(torch.float8_e4m3fn)
    scale = pool.view(torch.float32)[..., PAGE * d // 4]
    kv = [codes[i].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scale[i][table][..., None] for i in range(2)]
    k = kv[0].unflatten(3, (PAGE, d)).permute(0, 2, 4, 1, 3).reshape(B, hkv, d, L)
    v = kv[1].unflatten(3, (d, PAGE)).permute(0, 2, 1, 4, 3).reshape(B, hkv, L, d)
    s = (q.float().unflatten(1, (hkv, H // hkv)) * d ** -0.5) @ k                       # [B, hkv, g, L]
    s = s.masked_fill((torch.arange(L, device=q.device) >= lens[:, None])[:, None, None], float("-inf"))
    p = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    return ((p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)).reshape(B, H, d).to(q.dtype)


def _select(state):
    logits, scores, finished, n, pad = state["logits"], state["scores"], state["finished"], state["case"]["best"], 2
    if own:
        return _ops().beam_select(logits, scores, n, finished=finished, pad_token=pad)
    B, K = scores.shape
    # 64 bits: candidates of different beams are told apart by less than 32 bits of a logarithm of 150 thousand terms keep
    x = logits.double().unflatten(0, (B, K))
    x = x - x.amax(-1, keepdim=True)
    value = scores.double()[..., None] + (x - x.exp().sum(-1, keepdim=True).log())
    if finished is not None:
        only = torch.arange(x.shape[-1], device=x.device) == pad
        value = torch.where(finished[..., None], torch.where(only, scores.double()[..., None], float("-inf")), value)
    value, at = value.flatten(1).sort(dim=1, descending=True, stable=True)
    value, at = value[:, :n], at[:, :n]
    parent = at // x.shape[-1]
    return value.float(), (parent + K * torch.arange(B, device=x.device)[:, None]).int(), at - parent * x.shape[-1]


def _reorder(state):
    if own:
        state["reorder"](state["parents"])
    else:
        table, pool, parents, lens = state["table"], state["pool"], state["parents"].long(), state["lens"].long()
        full = lens // PAGE
        column = torch.arange(table.shape[1], device=table.device)
        # the open page of a row is its own: it gets the parent's bytes; a row that has none, or is its own parent, copies its page onto itself
        at = full.clamp_max(table.shape[1] - 1)[:, None]
        own_page = table.long().gather(1, at)[:, 0]
        theirs = table.long()[parents].gather(1, at)[:, 0]
        source = torch.where(lens % PAGE > 0, theirs, own_page)
        table.copy_(torch.where(column < full[:, None], table[parents], table))
        pool[:, :, own_page] = pool[:, :, source]
    return state["table"], state["pool"]


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "attention":
        return _exact_attention(s)
    if case["op"] == "select":
        return _exact_select(s)
    return None


def _e4m3(x):
    """Nearest e4m3 value of |x| <= 448, ties to even, in 64 bits."""
    step = torch.exp2((torch.frexp(x)[1] - 1).clamp_min(-6).double() - 3)
    return (x / step).round() * step


def _exact_append(s):
    q, lens = s["q"].double(), s["lens"].tolist()
    B, T, H, d = q.shape
    pool, hkv = s["pool"], s["k"].shape[2]
    half = d // 2
    out, turned = {}, []
    for x in (q, s["k"].double()):
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous())
        for b in range(B):
            z[b] *= torch.complex(s["cos"][lens[b]:lens[b] + T].double(), s["sin"][lens[b]:lens[b] + T].double())[:, None]
        turned.append(torch.cat((z.real, z.imag), -1))
    out["q"] = turned[0]
    for side, name, x in ((0, "k", turned[1]), (1, "v", s["v"].double())):
        codes = pool[side, :, :, :PAGE * d].view(torch.float8_e4m3fn).double()
        codes = codes.unflatten(2, (PAGE, d)) if side == 0 else codes.unflatten(2, (d, PAGE)).transpose(2, 3)
        codes = codes.contiguous()
        scale = pool[side].view(torch.float32)[:, :, PAGE * d // 4].double()
        for b in range(B):
            c, first = lens[b] % PAGE, lens[b] // PAGE
            n = (c + T + PAGE - 1) // PAGE
            ids = s["table"][b, first:first + n].long()
            room = torch.zeros(n * PAGE, hkv, d, dtype=torch.float64, device=x.device)
            room[c:c + T] = x[b]
            room = room.unflatten(0, (n, PAGE)).transpose(1, 2)                          # [n, hkv, 16, d]
            most = room.abs().amax((2, 3))
            bits = torch.log2(most.clamp_min(1e-300) / 448).ceil()
            bits = torch.where(most <= 448 * torch.exp2(bits - 1), bits - 1, bits)         # a logarithm may be off in its last place
            new = torch.exp2(bits.clamp(EXP_LO, EXP_HI))
            if c:
                new[0] = torch.maximum(new[0], scale[ids[0]])
                room[0, :, :c] = codes[ids[0], :, :c] * scale[ids[0]][:, None, None]
            codes[ids] = _e4m3((room / new[..., None, None]).clamp(-448, 448))
            scale[ids] = new
        codes = codes if side == 0 else codes.transpose(2, 3)
        out[name], out[name + "_scale"] = codes.reshape(codes.shape[0], hkv, PAGE * d), scale
    return {k: out[k] for k in ("q", "k", "k_scale", "v", "v_scale")}


def _exact_attention(s):
    q, lens = s["q"].double(), s["lens"].tolist()
    B, H, d = q.shape
    hkv = s["pool"].shape[2]
    out = torch.zeros_like(q)
    for b in range(B):
        n = (lens[b] + PAGE - 1) // PAGE
        if not n:
            continue
        ids = s["table"][b, :n].long()
        k, v = (s["pool"][i][ids] for i in range(2))
        ks, vs = (x.view(torch.float32)[..., PAGE * d // 4].double() for x in (k, v))
        k = k[..., :PAGE * d].contiguous().view(torch.float8_e4m3fn).double().reshape(n, hkv, PAGE, d) * ks[..., None, None]
        v = v[..., :PAGE * d].contiguous().view(torch.float8_e4m3fn).double().reshape(n, hkv, d, PAGE) * vs[..., None, None]
        k = k.transpose(0, 1).reshape(hkv, n * PAGE, d)[:, :lens[b]]
        v = v.permute(1, 0, 3, 2).reshape(hkv, n * PAGE, d)[:, :lens[b]]
        weight = torch.softmax(torch.einsum("hgd,hld->hgl", q[b].reshape(hkv, -1, d), k) / math.sqrt(d), -1)
        out[b] = torch.einsum("hgl,hld->hgd", weight, v).reshape(H, d)
    return out


def _exact_select(s):
    B, K = s["scores"].shape
    best = []
    for b in range(B):
        rows = torch.log_softmax(s["logits"][b * K:(b + 1) * K].double(), -1) + s["scores"][b].double()[:, None]
        if s["finished"] is not None:
            rows[s["finished"][b]] = float("-inf")
            rows[s["finished"][b], 2] = s["scores"][b].double()[s["finished"][b]]
        best.append(rows.flatten().topk(s["case"]["best"])[0])
    return torch.stack(best), None, None
