"""GPU: log probabilities, entropy, ranks and top tokens against 64 bits."""
import numpy as np
import pytest

import oracle.oracle as orc
import willamette_hip as wh
from device_arrays import Array, Graph, from_kind, to_kind

pytestmark = pytest.mark.gpu


def reference(x, tok, k):
    """x [rows, vocab] in 64 bits."""
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1, keepdims=True)
        base = np.where(np.isinf(m) & (m < 0), 0, m)
        e = np.exp(x - base)
        total = e.sum(1, keepdims=True)
        lp = np.where(total > 0, x - base - np.log(total), np.where(np.isnan(total), np.nan, -np.inf))
        p = e / total
        ent = -np.where(p > 0, p * lp, 0 * p).sum(1)
        ent = np.where(total[:, 0] == 0, 0, ent)
    bad = np.isnan(x).any(1) | np.isposinf(x).any(1)
    lp[bad], ent[bad] = np.nan, np.nan
    order = np.stack([np.lexsort((np.arange(x.shape[1]), -np.where(np.isnan(r), -np.inf, r), np.isnan(r))) for r in x])
    rank = np.array([-1 if not 0 <= t < x.shape[1] else int(np.where(o == t)[0][0]) for o, t in zip(order, tok)])
    at = np.array([np.nan if not 0 <= t < x.shape[1] else r[t] for r, t in zip(lp, tok)])
    top = order[:, :k]
    return at, ent, rank, top, np.take_along_axis(lp, top, 1)


def score(ctx, x, kind, first, stride, rows, vocab, tok, k, out, work, need):
    """One call; out: arrays of logprob, entropy, rank, top ids, top logprobs, or None."""
    ctx.check(wh.lib.wm_token_logprobs_dev(ctx.h, wh.DTYPES[kind], x.ptr + first * x.dtype.itemsize, stride, rows, vocab,
                                           None if tok is None else tok.ptr, k, *[None if o is None else o.ptr for o in out],
                                           work.ptr, need))


def outputs(ctx, rows, k):
    return [Array(ctx, np.full(s, 7, t)) for s, t in ((rows, np.float32), (rows, np.float32), (rows, np.int32),
                                                      ((rows, max(k, 1)), np.int32), ((rows, max(k, 1)), np.float32))]


def run(ctx, x, tok, k, kind="f32", first=0, stride=None):
    """x [rows, vocab] of a type; `first` and `stride`: where its rows lie in the device's buffer."""
    rows, vocab = x.shape
    stride = stride or vocab
    buf = np.full(first + rows * stride, to_kind(np.nan, kind))  # what is between the rows is not looked at
    np.lib.stride_tricks.as_strided(buf[first:], (rows, vocab), (stride * buf.itemsize, buf.itemsize))[:] = x
    need = wh.token_logprobs_workspace(rows, vocab, k)
    work = Array(ctx, np.full(max(need, 4) // 4, np.nan, np.float32))
    out = outputs(ctx, rows, k)
    d, t = Array(ctx, buf, kind), Array(ctx, tok)
    score(ctx, d, kind, first, stride, rows, vocab, t, k, out[:3] + (out[3:] if k else [None, None]), work, need)
    got = [o.host() for o in out]
    return got[:3] + [g[:, :k] for g in got[3:]]


def close(got, want, size):
    """f32 sums of `n` terms in trees and chains no longer than 2^10 steps, each exponential of an argument rounded
    to f32 (|x - m| up to `size`): the sum's relative error is under 2^-24 (2^10 + 4 + size); the logarithm and the
    differences add a step of their values."""
    tol = 2.0 ** -24 * (2 ** 10 + 16 + 4 * size) + 2.0 ** -23 * np.abs(want)
    ok = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    return bool(np.all(ok))


def check(got, x, tok, k):
    with np.errstate(invalid="ignore"):
        want = reference(x, tok, k)
        fin = x[np.isfinite(x)]
        size = min(120.0, float(np.ptp(fin))) if fin.size else 0.0
    assert np.array_equal(got[2], want[2])
    assert np.array_equal(got[3], want[3])
    assert close(got[0], want[0], size) and close(got[1], want[1], size * 4) and close(got[4], want[4], size)


@pytest.mark.parametrize("kind,rows,vocab,k", [
    ("f32", 1, 1, 1), ("f32", 3, 2, 2), ("f32", 2, 63, 63), ("f32", 1, 64, 64), ("f32", 5, 257, 20), ("f32", 4, 1000, 0),
    ("f32", 1, 128256, 20), ("f32", 2, 128256, 64), ("f32", 40, 4097, 5), ("f16", 7, 5003, 33), ("bf16", 1, 50257, 20),
    ("bf16", 300, 1031, 64), ("f16", 1, 131, 3), ("bf16", 70, 32001, 1), ("f32", 300, 9999, 2)])
def test_logprobs(ctx, kind, rows, vocab, k):
    rng = np.random.default_rng(rows * 7 + vocab + k)
    x = to_kind(rng.standard_normal((rows, vocab)) * 3, kind)
    h = from_kind(x, kind)
    tok = rng.integers(0, vocab, rows).astype(np.int32)
    tok[::3] = h.argmax(1)[::3]
    # rows that begin at any element: an odd first one, an odd stride
    check(run(ctx, x, tok, k, kind, 1, vocab + 3), h, tok, k)
    check(run(ctx, x, tok, k, kind), h, tok, k)


def test_logprobs_ties_take_the_lowest_id(ctx):
    rng = np.random.default_rng(1)
    x = rng.integers(-3, 4, (6, 3001)).astype(np.float32)
    x[1] = 2.0
    x[2, :] = np.where(rng.random(3001) < 0.5, 0.0, -0.0)  # one value
    tok = np.array([0, 1500, 3000, 77, 2999, 5], np.int32)
    got = run(ctx, x, tok, 64)
    check(got, x.astype(np.float64), tok, 64)
    assert np.array_equal(got[3][1], np.arange(64)) and got[2][1] == 1500


@pytest.mark.parametrize("order", ["rising", "falling"])
@pytest.mark.parametrize("vocab", [5000, 128256])
def test_logprobs_of_sorted_rows(ctx, order, vocab):
    """Every value passes the one before: the worst order for a running list."""
    x = np.linspace(-40, 30, vocab, dtype=np.float32)[None].repeat(2, 0)
    x = x if order == "rising" else x[:, ::-1].copy()
    tok = np.array([vocab // 2, 1], np.int32)
    check(run(ctx, x, tok, 64), x.astype(np.float64), tok, 64)


def test_logprobs_masked_and_not_numbers(ctx):
    rng = np.random.default_rng(2)
    vocab, inf = 2003, np.inf
    x = (rng.standard_normal((12, vocab)) * 3).astype(np.float32)
    x[0, 5:] = -inf                      # a mask that leaves five
    x[1] = -inf                          # one that leaves nothing
    x[2] = -inf
    x[2, 700] = -3.0                     # one
    x[3, 11] = np.nan
    x[4, 12] = inf
    x[5, 13], x[5, 14] = inf, np.nan
    x[6] = np.nan
    x[7] = np.finfo(np.float32).min      # the lowest value as a mask
    x[7, 9] = 1.0
    x[8] = np.finfo(np.float32).min
    x[9] = 3e38                          # equal and huge
    x[10, :] = -1e30
    x[11, 1000] = 3.4e38
    tok = np.array([700, 3, 700, 11, 12, 13, 0, 9, 4, 1, 2, 1000], np.int32)
    check(run(ctx, x, tok, 20), x.astype(np.float64), tok, 20)


def test_logprobs_tokens_outside_the_vocabulary(ctx):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 100)).astype(np.float32)
    tok = np.array([-1, 100, 1 << 30, 99], np.int32)
    got = run(ctx, x, tok, 2)
    check(got, x.astype(np.float64), tok, 2)
    assert np.isnan(got[0][:3]).all() and np.array_equal(got[2][:3], [-1, -1, -1])


def test_logprobs_outputs_one_at_a_time(ctx):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((3, 40000)).astype(np.float32)
    tok = np.array([5, 6, 7], np.int32)
    whole = run(ctx, x, tok, 7)
    need = wh.token_logprobs_workspace(3, 40000, 7)
    work, d, t = Array(ctx, np.zeros(max(need, 1), np.uint8)), Array(ctx, x, "f32"), Array(ctx, tok)
    for i in range(5):
        out = outputs(ctx, 3, 7)[i]
        score(ctx, d, "f32", 0, 40000, 3, 40000, t if i in (0, 2) else None, 7 if i >= 3 else 0,
              [out if j == i else None for j in range(5)], work, need)
        assert np.array_equal(out.host(), whole[i])


def test_logprobs_host_form_and_the_lm_head(ctx):
    """Scores of the lm-head's own logits: the argmax has rank 0 and leads the list."""
    rng = np.random.default_rng(5)
    raw = wh.synth_q6k(3, 4, 3000, 256)
    w = ctx.upload_q6k(raw, 256, 3000)
    hidden = rng.standard_normal((4, 256)).astype(np.float32)
    logits = np.stack([wh.compute_logits(ctx, w, h) for h in hidden])
    ids = np.array([orc.argmax(r) for r in logits], np.int32)
    got = wh.token_logprobs(ctx, logits, ids, 5)
    assert np.array_equal(got["rank"], [0, 0, 0, 0]) and np.array_equal(got["top_ids"][:, 0], ids)
    assert np.array_equal(got["top_logprobs"][:, 0], got["logprob"])
    check((got["logprob"], got["entropy"], got["rank"], got["top_ids"], got["top_logprobs"]),
          logits.astype(np.float64), ids, 5)
    assert set(wh.token_logprobs(ctx, logits)) == {"entropy"}
    w.close()


def test_logprobs_captured(ctx):
    rng = np.random.default_rng(6)
    x, tok = Array(ctx, np.zeros((2, 60000), np.float32), "f32"), Array(ctx, np.zeros(2, np.int32))
    out = outputs(ctx, 2, 9)
    need = wh.token_logprobs_workspace(2, 60000, 9)
    work = Array(ctx, np.zeros(max(need, 1), np.uint8))

    def call():
        score(ctx, x, "f32", 0, 60000, 2, 60000, tok, 9, out, work, need)
    g = Graph(ctx, call)
    for turn in range(4):
        h = (rng.standard_normal((2, 60000)) * 3).astype(np.float32)
        t = rng.integers(0, 60000, 2).astype(np.int32)
        x.put(h)
        tok.put(t)
        g.replay()
        first = [o.host() for o in out]
        check(first, h.astype(np.float64), t, 9)
        call()
        assert all(np.array_equal(a, o.host()) for a, o in zip(first, out))
    g.close()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("low", ["-inf", "lowest"])
def test_logprobs_of_masked_vocabularies(ctx, kind, low):
    """A grammar's mask leaves few tokens of a long row: none in most of its parts, all in one, some at the end."""
    rng = np.random.default_rng(7)
    vocab = 70001
    low = -np.inf if low == "-inf" else float(np.finfo(np.float32).min) if kind == "f32" else -3.3895314e38
    x = np.full((6, vocab), low, np.float32)
    x[0, [5, 40000, 70000]] = [1.0, 2.0, 3.0]
    x[1, 20000:20040] = rng.standard_normal(40)
    x[2, -700:] = rng.standard_normal(700)        # behind the mask
    x[3, 200:900] = 0.0                           # equal, and not at the beginning
    x[4, :64] = rng.standard_normal(64)
    x[5, ::300] = np.nan                          # no numbers, in each part
    x = to_kind(x, kind)
    tok = np.array([40000, 20001, 69000, 555, 65, 1], np.int32)
    for k in (64, 3):
        check(run(ctx, x, tok, k, kind), from_kind(x, kind), tok, k)


@pytest.mark.parametrize("kind,vocab", [("f32", 16 * 1024 + 5), ("f32", 65536 + 1), ("bf16", 16385), ("f16", 16384 + 600)])
def test_logprobs_with_a_short_last_part(ctx, kind, vocab):
    rng = np.random.default_rng(8)
    x = to_kind(rng.standard_normal((2, vocab)) * 3, kind)
    x[1, -1] = to_kind(20.0, kind)
    tok = np.array([vocab - 1, 3], np.int32)
    for k in (0, 64):
        check(run(ctx, x, tok, k, kind), from_kind(x, kind), tok, k)
        check(run(ctx, x.repeat(80, 0), tok.repeat(80), k, kind), from_kind(x, kind).repeat(80, 0), tok.repeat(80), k)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("k", [0, 4])
def test_logprobs_of_rows_that_rise_late_or_lie_far_out(ctx, kind, k):
    """Sums relative to a part's first values, where later ones are far above, below, or all are large."""
    rng = np.random.default_rng(9)
    x = (rng.standard_normal((6, 30000)) * 3).astype(np.float32)
    x[0, 25000:] += 60.0
    x[1, 9000] = 900.0
    x[2, 4000:] -= 500.0
    x[3] += 1e4
    x[4] = x[4] * 300 - 2e4
    x[5, :3000] = -np.inf
    x = to_kind(x, kind)
    tok = np.array([25001, 9000, 1, 77, 5, 2], np.int32)
    check(run(ctx, x, tok, k, kind), from_kind(x, kind), tok, k)


def test_logprobs_do_not_depend_on_what_else_is_asked(ctx):
    rng = np.random.default_rng(10)
    x = (rng.standard_normal((150, 70000)) * 3).astype(np.float32)
    x[3, 60000:] += 80.0
    tok = rng.integers(0, 70000, 150).astype(np.int32)
    a, b, one = run(ctx, x, tok, 0), run(ctx, x, tok, 9), run(ctx, x[3:4], tok[3:4], 0)
    assert all(np.array_equal(p, q) for p, q in zip(a[:3], b[:3]))
    assert one[2][0] == a[2][3]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_logprobs_in_the_workspace_of_a_larger_call(ctx, kind):
    """The workspace of many rows serves few, which are divided into more parts; nothing behind it is written."""
    rng = np.random.default_rng(11)
    rows, vocab, k = 60, 50001, 9
    size = wh.token_logprobs_workspace(rows, vocab, k)
    work = Array(ctx, np.full(size // 4 + 100, np.nan, np.float32))
    for n, v in ((rows, vocab), (32, vocab), (31, vocab), (1, vocab), (rows, 16385), (rows, 4097), (rows, 100), (128, 16000)):
        x = to_kind(rng.standard_normal((n, v)) * 3, kind)
        tok = rng.integers(0, v, n).astype(np.int32)
        out = outputs(ctx, n, k)
        if n <= rows:
            score(ctx, Array(ctx, x, kind), kind, 0, v, n, v, Array(ctx, tok), k, out, work, size)
            check([o.host() for o in out], from_kind(x, kind), tok, k)
            assert np.isnan(work.host()[size // 4:]).all()
        # its own size is enough too
        check(run(ctx, x, tok, k, kind), from_kind(x, kind), tok, k)


@pytest.mark.parametrize("kind,rows,vocab", [("f32", 3, 128256), ("f32", 200, 50257), ("f16", 200, 128256), ("bf16", 2, 9999)])
def test_logprobs_count_as_32_bits(ctx, kind, rows, vocab):
    """Log probabilities to what their own additions and exponentials may be off by.

    A lane adds up to 64 exponentials, 6 exchanges a wave, 3 additions the waves, 14 at most the parts: 87 roundings of
    2^-24.  An exponential is good to 2^-23, and its argument, up to r / ln 2 for logits r apart, to 2^-24 and the
    constant's 2^-26 of it: 2 + 1.25 r steps.  The sum's relative error is the logarithm's absolute one; the logarithm
    and two differences add two steps of at most twice the largest value."""
    rng = np.random.default_rng(12)
    x = to_kind(rng.standard_normal((rows, vocab)) * 3, kind)
    h = from_kind(x, kind)
    tok = rng.integers(0, vocab, rows).astype(np.int32)
    got = run(ctx, x, tok, 5, kind)
    want = reference(h, tok, 5)
    r = float(np.ptp(h))
    for i in (0, 4):
        assert np.all(np.abs(got[i] - want[i]) <= 2.0 ** -24 * (87 + 2 + 1.25 * r + 4 * 2 * np.abs(want[i])))
