"""Timing cases of the paged 8-bit KV cache and of token scoring: appending a
step's keys and values (rotated on the way), attention over the pages, the
pages' values read back, and the log probabilities of given tokens.

A case is a plain dict; `prepare` makes what a serving program holds before
the call (activations, the page pool, the step's page table and lengths, the
rotation's tables, logits), `run` makes one pass: in elementary torch
operations, or, with `own`, through the library's entry points.  Sizes are
BitNet-2B's (20 query heads over 5 kv heads of 128, 128256 tokens) and, in
drawn cases, those of smaller models and other vocabularies.

The cache, per layer: pages of `page` tokens; in a page, for each kv head,
K's codes [token][dim], V's codes [dim][token] and one f32 scale for K and V.
Token j of a sequence with n new tokens and a cache of L positions (the new
ones included) is at position L - n + j.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

# (query heads, kv heads): BitNet-2B, and smaller models of the same build
HEADS = {"2b": (20, 5), "1b": (16, 4), "small": (8, 2)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of a small batch: one token of each of 16 sequences
        {"name": "append_decode_16", "kind": "append", "type": "f32", "heads": "2b", "dim": 128, "page": 16,
         "n_seqs": 16, "ctx_lo": 128, "ctx_hi": 4064, "new_lo": 1, "new_hi": 1, "n_rot": 128, "layout": "half"},
        # a continuous-batching step: decoding sequences and prompt chunks
        {"name": "append_ragged_24", "kind": "append", "type": "bf16", "heads": "2b", "dim": 128, "page": 64,
         "n_seqs": 24, "ctx_lo": 0, "ctx_hi": 4064, "new_lo": 1, "new_hi": 100, "n_rot": 64,
         "layout": "interleaved"},
        # eight prompts of different lengths, packed, into empty caches
        {"name": "append_prompts_8", "kind": "append", "type": "f32", "heads": "2b", "dim": 128, "page": 16,
         "n_seqs": 8, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 100, "new_hi": 2000, "n_rot": 128, "layout": "half"},
        # one token of one chat of 1024 positions: latency
        {"name": "attention_decode_1", "kind": "attention", "type": "f32", "heads": "2b", "dim": 128, "page": 16,
         "n_seqs": 1, "ctx_lo": 1023, "ctx_hi": 1023, "new_lo": 1, "new_hi": 1},
        # a decode step of 16 sequences of very different lengths
        {"name": "attention_decode_16", "kind": "attention", "type": "f32", "heads": "2b", "dim": 128, "page": 16,
         "n_seqs": 16, "ctx_lo": 128, "ctx_hi": 4064, "new_lo": 1, "new_hi": 1},
        # a decode step of a full server, long documents
        {"name": "attention_decode_64_long", "kind": "attention", "type": "bf16", "heads": "2b", "dim": 128,
         "page": 64, "n_seqs": 64, "ctx_lo": 2000, "ctx_hi": 16000, "new_lo": 1, "new_hi": 1},
        # a continuous-batching step: 1 to 32 new tokens of each sequence
        {"name": "attention_ragged_16", "kind": "attention", "type": "f32", "heads": "2b", "dim": 128, "page": 16,
         "n_seqs": 16, "ctx_lo": 128, "ctx_hi": 4064, "new_lo": 1, "new_hi": 32},
        # eight whole prompts of different lengths, packed
        {"name": "attention_prompts_8", "kind": "attention", "type": "f16", "heads": "2b", "dim": 128, "page": 32,
         "n_seqs": 8, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 100, "new_hi": 2000},
        # one long prompt
        {"name": "attention_prompt_8192", "kind": "attention", "type": "bf16", "heads": "2b", "dim": 128, "page": 64,
         "n_seqs": 1, "ctx_lo": 0, "ctx_hi": 0, "new_lo": 8192, "new_hi": 8192},
        # the sampled token's score and its alternatives, one chat
        {"name": "logprobs_1", "kind": "logprobs", "type": "f32", "rows": 1, "vocab": 128256, "top_k": 20},
        # every token of a prompt scored
        {"name": "logprobs_prompt_512", "kind": "logprobs", "type": "f32", "rows": 512, "vocab": 128256, "top_k": 5},
        # perplexity of a text under half-width logits, an odd vocabulary
        {"name": "logprobs_text_2047", "kind": "logprobs", "type": "bf16", "rows": 2047, "vocab": 50257, "top_k": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "logprobs", "logprobs"])
    c = {"kind": kind, "type": rng.choice(sorted(TYPES))}
    if kind == "logprobs":
        c.update(rows=_log(rng, 1, 400), vocab=_log(rng, 2000, 152000), top_k=rng.choice([0, 1, 5, 20, rng.randint(2, 64)]))
        return c
    c.update(heads=rng.choice(sorted(HEADS)), dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64]))
    mode = rng.choice(["decode", "ragged", "prompts"])
    if mode == "decode":
        lo = _log(rng, 1, 4000)
        c.update(n_seqs=_log(rng, 1, 48), ctx_lo=lo, ctx_hi=rng.randint(lo, 8000), new_lo=1, new_hi=1)
    elif mode == "ragged":
        lo = _log(rng, 1, 2000)
        c.update(n_seqs=rng.randint(2, 24), ctx_lo=lo, ctx_hi=rng.randint(lo, 5000), new_lo=1,
                 new_hi=_log(rng, 2, 200))
    else:
        lo = _log(rng, 2, 1200)
        c.update(n_seqs=rng.randint(1, 6), ctx_lo=0, ctx_hi=rng.choice([0, _log(rng, 16, 1000)]), new_lo=lo,
                 new_hi=rng.randint(lo, 1500))
    if kind == "append":
        c.update(n_rot=rng.choice([c["dim"], c["dim"], c["dim"] // 2, 48]), layout=rng.choice(["half", "interleaved"]))
    return c


# --- inputs ----------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed & 0x7FFFFFFFFFFFFFFF)
    return g


def _lengths(case):
    """(positions before, new tokens) of each sequence: fixed by the case."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    return [(r.randint(case["ctx_lo"], case["ctx_hi"]), r.randint(case["new_lo"], case["new_hi"]))
            for _ in range(case["n_seqs"])]


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _cum(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _layout(case, g):
    """The step's lengths and page table: pages in no order, a tenth of the pool free."""
    steps = _lengths(case)
    page = case["page"]
    used = [-(-(c + n) // page) for c, n in steps]
    n_pages = sum(used) + max(1, sum(used) // 10)
    perm = torch.randperm(n_pages, device="cuda", generator=g).cpu().tolist()
    width, at, table = max(used), 0, []
    for u in used:
        table.append(perm[at:at + u] + [0] * (width - u))
        at += u
    return {"case": case, "kind": case["kind"], "page": page, "n_pages": n_pages, "n_seqs": len(steps),
            "n_tokens": sum(n for _, n in steps), "max_new": max(n for _, n in steps),
            "max_kv": max(c + n for c, n in steps), "cu": _ints(_cum([n for _, n in steps])),
            "kv_len": _ints([c + n for c, n in steps]), "table": _ints(table)}


def _pool(st, case, g):
    """Codes as a quantiser leaves them, scales of blocks of about unit-size values."""
    _, kh = HEADS[case["heads"]]
    n, page, dim = st["n_pages"], case["page"], case["dim"]
    for name, shape in (("k", (n, kh, page, dim)), ("v", (n, kh, dim, page))):
        codes = torch.empty(shape, dtype=torch.int8, device="cuda")
        for part in codes.split(max(1, (1 << 26) // (kh * page * dim))):
            part.copy_((torch.randn(part.shape, device="cuda", generator=g) * 36).round_().clamp_(-127, 127))
        st[name + "_codes"] = codes
        st[name + "_scale"] = torch.exp(torch.randn(n, kh, device="cuda", generator=g) * 0.25) / 36


def _tables(n_pos, n_rot, base=500000.0):
    """The rotation's cosines and sines, angles in 64 bits."""
    inv = base ** (-torch.arange(0, n_rot, 2, dtype=torch.float64, device="cuda") / n_rot)
    a = torch.arange(n_pos, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    kind, g, dt = case["kind"], _gen(seed), TYPES[case["type"]]
    if kind == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.empty(rows, vocab, dtype=dt, device="cuda")
        for part in x.split(max(1, (1 << 26) // vocab)):
            v = torch.randn(part.shape, device="cuda", generator=g) * 2.0
            top = torch.randint(0, vocab, (part.shape[0], 40), device="cuda", generator=g)
            v.scatter_add_(1, top, torch.rand(top.shape, device="cuda", generator=g) * 8.0 + 4.0)
            part.copy_(v)
        # what was said: often the likeliest token, sometimes any
        tok = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.6, x.argmax(1),
                          torch.randint(0, vocab, (rows,), device="cuda", generator=g)).int()
        k = case["top_k"]
        return {"case": case, "kind": kind, "x": x, "tok": tok, "logprob": torch.empty(rows, device="cuda"),
                "entropy": torch.empty(rows, device="cuda"), "rank": torch.empty(rows, dtype=torch.int32, device="cuda"),
                "top_ids": torch.empty(rows, k, dtype=torch.int32, device="cuda"),
                "top_logprobs": torch.empty(rows, k, device="cuda")}
    st = _layout(case, g)
    _pool(st, case, g)
    (h, kh), dim, t = HEADS[case["heads"]], case["dim"], st["n_tokens"]
    if kind == "attention":
        # queries twice unit size: scores of standard deviation about 2
        st["q"] = (torch.randn(t, h, dim, device="cuda", generator=g) * 2.0).to(dt)
        st["out"] = torch.empty(t, h, dim, dtype=dt, device="cuda")
        st["lse"] = torch.empty(t, h, device="cuda")
        return st
    # the QKV projection's output, a few large channels among its keys
    qkv = torch.randn(t, (h + 2 * kh) * dim, device="cuda", generator=g)
    qkv *= torch.where(torch.rand(qkv.shape[1], device="cuda", generator=g) < 0.02, 4.0, 1.0)
    st["qkv"] = qkv.to(dt)
    st["q_out"] = torch.empty(t, h, dim, dtype=dt, device="cuda")
    st["cos"], st["sin"] = _tables(st["max_kv"], case["n_rot"])
    # the pages that the step writes, and every position that they then hold
    page, seq, lp, first, count = st["page"], [], [], [], []
    for s, (c, n) in enumerate(_lengths(case)):
        pages = range(c // page, (c + n - 1) // page + 1)
        seq += [s] * len(pages)
        lp += list(pages)
        count.append(c + n - c // page * page)
    st["w_seq"], st["w_lp"] = _ints(seq, torch.int64), _ints(lp, torch.int64)
    st["r_cu"], st["r_tokens"], st["r_max"] = _ints(_cum(count)), sum(count), max(count)
    st["k_out"] = torch.empty(st["r_tokens"], kh, dim, dtype=dt, device="cuda")
    st["v_out"] = torch.empty_like(st["k_out"])
    return st


# --- one pass, plain --------------------------------------------------------

def _positions(st, cu, n_tokens):
    """Sequence and position of every packed token."""
    t = torch.arange(n_tokens, device="cuda")
    s = torch.bucketize(t, cu[1:].long(), right=True)
    return s, st["kv_len"][s] - (cu[s + 1] - cu[s]) + (t - cu[s])


def _rotate(x, cos, sin, layout):
    """x [token, head, dim] in 64 bits, cos and sin [token, pair]."""
    n = 2 * cos.shape[1]
    c, s = cos[:, None].double(), sin[:, None].double()
    if layout == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., n:]], -1)


def _round(x):
    """To whole numbers, halves away from zero."""
    return torch.trunc(x + torch.copysign(torch.full_like(x, 0.5), x))


def _blocks(st, x, codes, scale):
    """The written pages' codes [page, token, head, dim] and scales [page, head] after the append of x
    [token, head, dim]; `codes` laid out the same, from before."""
    page, seq, lp = st["page"], st["w_seq"], st["w_lp"]
    ids = st["table"][seq, lp].long()
    pos = lp[:, None] * page + torch.arange(page, device="cuda")
    end = st["kv_len"][seq].long()[:, None]
    cu = st["cu"].long()
    start = end - (cu[seq + 1] - cu[seq])[:, None]
    new, old = (pos >= start) & (pos < end), pos < start
    tok = (cu[seq][:, None] + pos - start).clamp(0, x.shape[0] - 1)
    val = x[tok].float() * new[..., None, None]
    s_old = scale[ids] * old.any(1)[:, None]
    s_new = torch.maximum(s_old, (val.abs().amax((1, 3)).double() / 127.0).float())
    div = torch.where(s_new > 0, s_new, 1.0).double()[:, None, :, None]
    fresh = _round(val.double() / div).clamp_(-127, 127)
    kept = _round(codes.double() * s_old.double()[:, None, :, None] / div)
    out = torch.where(new[..., None, None], fresh, torch.where(old[..., None, None], kept, codes.double()))
    return ids, out.to(torch.int8), s_new


def _gather(st, codes, scale, s, pos):
    """Values of packed tokens: codes [page id, head, token, dim] times their block's scale."""
    ids = st["table"][s, (pos // st["page"])].long()
    return codes[ids, :, pos % st["page"]].float() * scale[ids][..., None]


def _append(st):
    case, dt = st["case"], TYPES[st["case"]["type"]]
    (h, kh), dim = HEADS[case["heads"]], case["dim"]
    _, pos = _positions(st, st["cu"], st["n_tokens"])
    cos, sin = st["cos"][pos], st["sin"][pos]
    q, k, v = st["qkv"].view(st["n_tokens"], h + 2 * kh, dim).split([h, kh, kh], 1)
    st["q_out"].copy_(_rotate(q.double(), cos, sin, case["layout"]))
    ids = st["table"][st["w_seq"], st["w_lp"]].long()
    ids, codes, scale = _blocks(st, _rotate(k.double(), cos, sin, case["layout"]), st["k_codes"][ids].transpose(1, 2),
                                st["k_scale"])
    st["k_codes"][ids] = codes.transpose(1, 2)
    st["k_scale"][ids] = scale
    ids, codes, scale = _blocks(st, v, st["v_codes"][ids].permute(0, 3, 1, 2), st["v_scale"])
    st["v_codes"][ids] = codes.permute(0, 2, 3, 1)
    st["v_scale"][ids] = scale
    s, pos = _positions(st, st["r_cu"], st["r_tokens"])
    return {"q": st["q_out"], "k": _gather(st, st["k_codes"], st["k_scale"], s, pos).to(dt),
            "v": _gather(st, st["v_codes"].transpose(2, 3), st["v_scale"], s, pos).to(dt)}


def _attention(st):
    case, dt = st["case"], TYPES[st["case"]["type"]]
    (h, kh), dim, n, t = HEADS[case["heads"]], case["dim"], st["n_seqs"], st["n_tokens"]
    ids = st["table"].long()
    length = ids.shape[1] * st["page"]
    k = (st["k_codes"][ids].float() * st["k_scale"][ids][..., None, None]).permute(0, 2, 4, 1, 3).reshape(n * kh, dim, length)
    s, pos = _positions(st, st["cu"], t)
    j = torch.arange(t, device="cuda") - st["cu"][s]
    m = st["max_new"]
    q = torch.zeros(n, m, h, dim, device="cuda")
    q[s, j] = st["q"].float()
    at = torch.full((n, m), -1, device="cuda", dtype=torch.int64)
    at[s, j] = pos
    q = q.view(n, m, kh, h // kh, dim).transpose(1, 2).reshape(n * kh, m * (h // kh), dim)
    x = torch.bmm(q, k).view(n, kh, m, h // kh, length) / math.sqrt(dim)
    x.masked_fill_(torch.arange(length, device="cuda") > at[:, None, :, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_min_(-3e38)
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    v = (st["v_codes"][ids].float() * st["v_scale"][ids][..., None, None]).permute(0, 2, 1, 4, 3).reshape(n * kh, length, dim)
    o = torch.bmm(x.view(n * kh, -1, length), v).view(n, kh, m, h // kh, dim) / total
    lse = (top + total.log())[..., 0]
    return {"out": o.transpose(1, 2)[s, j].reshape(t, h, dim).to(dt),
            "lse": lse.transpose(1, 2)[s, j].reshape(t, h)}


def _logprobs(st):
    vocab, tok, k = st["case"]["vocab"], st["tok"].long()[:, None], st["case"]["top_k"]
    x = st["x"].float()
    top = x.amax(1, keepdim=True)
    d = x - top
    e = d.exp()
    total = e.sum(1, keepdim=True)
    norm = top + total.log()
    xt = x.gather(1, tok)
    ids = torch.arange(vocab, device="cuda")
    out = {"logprob": (xt - norm)[:, 0], "entropy": (total.log() - (e * d).sum(1, keepdim=True) / total)[:, 0],
           "rank": ((x > xt) | ((x == xt) & (ids < tok))).sum(1).int()}
    if k:
        # values in order, equal ones by their index: a key of both
        bits = x.view(torch.int32)
        key = ((bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() << 32) | (0xFFFFFFFF - ids)
        out["top_ids"] = (0xFFFFFFFF - (key.topk(k, 1).values & 0xFFFFFFFF)).int()
        out["top_logprobs"] = x.gather(1, out["top_ids"].long()) - norm
    return out


# --- one pass, the library's -------------------------------------------------

_CTX = []


def _lib():
    """The library and the program's one context, whose stream torch then works on too, so that what either enqueues
    is in order; what torch had enqueued before is waited for."""
    if not _CTX:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "project-willamette_amd"))
        import willamette_hip as wh
        ctx = wh.Context(0)
        torch.cuda.synchronize()
        torch.cuda.set_stream(torch.cuda.ExternalStream(ctx.stream))
        _CTX.extend([wh, ctx])
    return _CTX


def _descriptors(st, wh):
    """The cache's and the step's descriptors, and the workspace: kept with the buffers they describe."""
    if "own" in st:
        return st["own"]
    case = st["case"]
    (h, kh), dim = HEADS[case["heads"]], case["dim"]
    kv = wh.PagedKV(st["k_codes"].data_ptr(), st["v_codes"].data_ptr(), st["k_scale"].data_ptr(),
                    st["v_scale"].data_ptr(), st["n_pages"], st["page"], kh, dim)

    def batch(cu, tokens, most):
        return wh.PagedBatch(cu.data_ptr(), st["kv_len"].data_ptr(), st["table"].data_ptr(), st["n_seqs"],
                             st["table"].shape[1], tokens, most, st["max_kv"])
    o = {"kv": kv, "batch": batch(st["cu"], st["n_tokens"], st["max_new"]), "type": wh.DTYPES[case["type"]]}
    if case["kind"] == "append":
        o["read"] = batch(st["r_cu"], st["r_tokens"], st["r_max"])
        o["rope"] = wh.Rope(st["cos"].data_ptr(), st["sin"].data_ptr(), st["max_kv"], case["n_rot"],
                            wh.ROPE_HALF if case["layout"] == "half" else wh.ROPE_INTERLEAVED)
    else:
        o["bytes"] = wh.paged_attention_workspace(kv, o["batch"], h)
        o["work"] = torch.empty(max(1, o["bytes"]), dtype=torch.uint8, device="cuda")
    st["own"] = o
    return o


def _run_own(st):
    wh, ctx = _lib()
    lib, case = wh.lib, st["case"]
    if st["kind"] == "logprobs":
        rows, vocab, k = case["rows"], case["vocab"], case["top_k"]
        if "work" not in st:
            st["bytes"] = wh.token_logprobs_workspace(rows, vocab, k)
            st["work"] = torch.empty(max(1, st["bytes"]), dtype=torch.uint8, device="cuda")
        ctx.check(lib.wm_token_logprobs_dev(
            ctx.h, wh.DTYPES[case["type"]], st["x"].data_ptr(), vocab, rows, vocab, st["tok"].data_ptr(), k,
            st["logprob"].data_ptr(), st["entropy"].data_ptr(), st["rank"].data_ptr(),
            st["top_ids"].data_ptr() if k else None, st["top_logprobs"].data_ptr() if k else None,
            st["work"].data_ptr(), st["bytes"]))
        out = {"logprob": st["logprob"], "entropy": st["entropy"], "rank": st["rank"]}
        return out | ({"top_ids": st["top_ids"], "top_logprobs": st["top_logprobs"]} if k else {})
    o = _descriptors(st, wh)
    (h, kh), dim = HEADS[case["heads"]], case["dim"]
    if st["kind"] == "attention":
        ctx.check(lib.wm_paged_attention_dev(
            ctx.h, o["kv"], o["batch"], o["type"], st["q"].data_ptr(), h * dim, h, 1.0 / math.sqrt(dim),
            st["out"].data_ptr(), h * dim, st["lse"].data_ptr(), o["work"].data_ptr(), o["bytes"]))
        return {"out": st["out"], "lse": st["lse"]}
    at, size, row = st["qkv"].data_ptr(), st["qkv"].element_size(), (h + 2 * kh) * dim
    ctx.check(lib.wm_paged_kv_append_dev(
        ctx.h, o["kv"], o["batch"], o["rope"], o["type"], at, row, h, at + h * dim * size, row,
        at + (h + kh) * dim * size, row, st["q_out"].data_ptr(), h * dim))
    ctx.check(lib.wm_paged_kv_read_dev(
        ctx.h, o["kv"], o["read"], o["type"], st["k_out"].data_ptr(), kh * dim, st["v_out"].data_ptr(), kh * dim))
    return {"q": st["q_out"], "k": st["k_out"], "v": st["v_out"]}


def run(st):
    if own:
        return _run_own(st)
    return {"append": _append, "attention": _attention, "logprobs": _logprobs}[st["kind"]](st)


# --- what a pass cannot do without ------------------------------------------

def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "logprobs":
        n, k = case["rows"] * case["vocab"], case["top_k"]
        return {"bytes": n * size + case["rows"] * (4 + 12 + 8 * k), "flops": 6 * n}
    (h, kh), dim, page = HEADS[case["heads"]], case["dim"], case["page"]
    nbytes = flops = 0
    for c, n in _lengths(case):
        pages = -(-(c + n) // page)
        if case["kind"] == "attention":
            nbytes += 2 * kh * ((c + n) * dim + 4 * pages) + 2 * n * h * dim * size + 4 * n * h + 4 * pages + 8
            flops += 4 * h * dim * (n * c + n * (n + 1) // 2)
        else:
            old = c % page                    # tokens of the first page that were there
            touched = pages - c // page
            nbytes += n * dim * size * (2 * h + 2 * kh) + 2 * kh * dim * (2 * old + n) + 16 * kh * touched
            nbytes += 4 * n * case["n_rot"]   # cosines and sines
            nbytes += 2 * kh * dim * (old + n) * size  # read back; the codes are where the append left them
            flops += 3 * n * case["n_rot"] * (h + kh) + 6 * (n + old) * kh * dim
    return {"bytes": nbytes, "flops": flops}


# --- the same in 64 bits ------------------------------------------------------

def _exact_attention(st, case):
    (h, kh), dim = HEADS[case["heads"]], case["dim"]
    outs, lses, at = [], [], 0
    for s, (c, n) in enumerate(_lengths(case)):
        used = -(-(c + n) // case["page"])
        ids = st["table"][s, :used].long()
        k = st["k_codes"][ids].double() * st["k_scale"][ids].double()[..., None, None]
        v = st["v_codes"][ids].double() * st["v_scale"][ids].double()[..., None, None]
        k = k.permute(1, 3, 0, 2).reshape(kh, 1, dim, -1)[..., :c + n].contiguous()
        v = v.permute(1, 0, 3, 2).reshape(kh, 1, -1, dim)[:, :, :c + n].contiguous()
        q = st["q"][at:at + n].double().view(n, kh, h // kh, dim).permute(1, 2, 0, 3).contiguous()
        x = torch.matmul(q, k) * dim ** -0.5
        x += torch.full((n, c + n), -math.inf, dtype=torch.float64, device="cuda").triu_(c + 1)
        z = torch.logsumexp(x, -1)
        x.sub_(z[..., None]).exp_()
        outs.append(torch.matmul(x, v).permute(2, 0, 1, 3).reshape(n, h, dim))
        lses.append(z.permute(2, 0, 1).reshape(n, h))
        at += n
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_block(rows, old_codes, s_old):
    """One block of one head: its values after `rows` [n, dim] (32 bits) join `old_codes` [m, dim]."""
    s = max(s_old, float((rows.abs().amax() / 127.0).float())) if rows.numel() else s_old
    q = torch.cat([old_codes * s_old, rows]) / s
    return torch.where(q < 0, (q - 0.5).ceil(), (q + 0.5).floor()).clamp(-127, 127) * s


def _exact_append(st, case):
    (h, kh), dim, page, pairs = HEADS[case["heads"]], case["dim"], case["page"], case["n_rot"] // 2
    q, k, v = st["qkv"].view(-1, h + 2 * kh, dim).double().cpu().split([h, kh, kh], 1)
    cos, sin = st["cos"].double().cpu(), st["sin"].double().cpu()
    table, kc, vc = st["table"].cpu().tolist(), st["k_codes"].cpu(), st["v_codes"].cpu()
    ks, vs = st["k_scale"].cpu().double(), st["v_scale"].cpu().double()
    pick = torch.arange(2 * pairs).view(2, pairs).t() if case["layout"] == "half" else torch.arange(2 * pairs).view(pairs, 2)

    def turned(x, c, n):
        y = x.clone()
        z = torch.complex(x[..., pick[:, 0]], x[..., pick[:, 1]]) * torch.complex(cos[c:c + n], sin[c:c + n])[:, None]
        y[..., pick[:, 0]], y[..., pick[:, 1]] = z.real, z.imag
        return y

    out, at = {"q": [], "k": [], "v": []}, 0
    for s, (c, n) in enumerate(_lengths(case)):
        out["q"].append(turned(q[at:at + n], c, n))
        kr, vr = turned(k[at:at + n], c, n).float().double(), v[at:at + n]
        for lp in range(c // page, (c + n - 1) // page + 1):
            b, m = table[s][lp], max(0, min(page, c - lp * page))
            lo, hi = max(0, lp * page - c), min(n, (lp + 1) * page - c)
            for name, x, codes, scale in (("k", kr, kc[b], ks[b]), ("v", vr, vc[b].transpose(1, 2), vs[b])):
                heads = [_exact_block(x[lo:hi, i], codes[i, :m].double(), float(scale[i]) if m else 0.0) for i in range(kh)]
                out[name].append(torch.stack(heads, 1))
        at += n
    return {name: torch.cat(x).cuda() for name, x in out.items()}


def _exact_logprobs(st, case):
    k, tok = case["top_k"], st["tok"].long()
    parts = []
    for x, t in zip(st["x"].split(256), tok.split(256)):
        p = torch.log_softmax(x.double(), 1)
        parts.append((p.gather(1, t[:, None])[:, 0], -(p.exp() * p).sum(1),
                      p.topk(k, 1).values))
    lp, ent, top = (torch.cat(v) for v in zip(*parts))
    out = {"logprob": lp, "entropy": ent, "rank": None}
    return out | ({"top_ids": None, "top_logprobs": top} if k else {})


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["kind"]](st, case)
