"""GPU: the paged 8-bit KV cache (append with rotation, read back, attention)
against the same in 64 bits (paged_ref.py)."""
import numpy as np
import pytest

import paged_ref as ref
import willamette_hip as wh
from device_arrays import Array, Graph, to_kind, typed
from paged_ref import Step

pytestmark = pytest.mark.gpu


def tables(n_pos, n_rot, base=10000.0):
    a = np.arange(n_pos)[:, None] * base ** (-np.arange(0, n_rot, 2) / max(n_rot, 1))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rope_of(ctx, cos, sin, n_rot, layout):
    """A rotation's descriptor, and the arrays it points to."""
    a, b = Array(ctx, cos), Array(ctx, sin)
    return wh.Rope(a.ptr, b.ptr, len(cos), n_rot, layout), a, b


class Device:
    """A step and its pool on the device, and the calls on them.  Packed arrays are (Array, row stride, first
    element), or an Array of [tokens, heads, dim] alone."""

    def __init__(self, ctx, st, pool):
        self.ctx, self.st = ctx, st
        self.pool = [Array(ctx, x) for x in pool]
        self.cu, self.len, self.table = Array(ctx, st.cu), Array(ctx, st.kv_len), Array(ctx, st.table)
        self.kv = wh.PagedKV(*[x.ptr for x in self.pool], st.n_pages, st.page, st.kh, st.dim)
        self.b = wh.PagedBatch(self.cu.ptr, self.len.ptr, self.table.ptr, len(st.steps), st.stride, st.n_tokens,
                               st.max_new, st.max_kv)

    @staticmethod
    def at(x):
        """Address and row stride."""
        if x is None:
            return None, 0
        x, stride, first = x if isinstance(x, tuple) else (x, int(np.prod(x.shape[1:])), 0)
        return x.ptr + first * x.dtype.itemsize, stride

    def append(self, kind, q, k, v, q_out, rope=None, heads=None):
        heads = heads if heads is not None else q.shape[1] if q is not None else 0
        self.ctx.check(wh.lib.wm_paged_kv_append_dev(self.ctx.h, self.kv, self.b, rope, wh.DTYPES[kind], *self.at(q),
                                                     heads, *self.at(k), *self.at(v), *self.at(q_out)))

    def read(self, kind, k, v):
        self.ctx.check(wh.lib.wm_paged_kv_read_dev(self.ctx.h, self.kv, self.b, wh.DTYPES[kind], *self.at(k), *self.at(v)))

    def attend(self, kind, q, out, lse, scale, work=None, heads=None):
        heads = heads or q.shape[1]
        need = wh.paged_attention_workspace(self.kv, self.b, heads)
        if work is None:
            # full of NaN: nothing may be read that was not written
            self.work = work = Array.full(self.ctx, (max(need, 4) // 4,), np.nan, "f32")
        q, qs = self.at(q)
        self.ctx.check(wh.lib.wm_paged_attention_dev(self.ctx.h, self.kv, self.b, wh.DTYPES[kind], q, qs, heads, scale,
                                                     *self.at(out), None if lse is None else lse.ptr, work.ptr, need))

    def host_pool(self):
        return [x.host() for x in self.pool]


def same_bits(a, b):
    a, b = np.asarray(a), np.asarray(b)
    return a.shape == b.shape and a.dtype == b.dtype and a.tobytes() == b.tobytes()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

# type, page, kv heads, group, dim, n_rot, layout, steps
APPENDS = [
    ("f32", 16, 5, 4, 128, 128, wh.ROPE_HALF, [(0, 1)]),
    ("f32", 16, 5, 4, 128, 128, wh.ROPE_HALF, [(37, 1), (15, 1), (16, 1), (0, 1), (31, 1)]),
    ("f32", 16, 2, 1, 64, 64, wh.ROPE_INTERLEAVED, [(3, 40), (0, 16), (16, 16), (30, 5), (9, 0), (12, 3)]),
    ("f16", 32, 3, 2, 128, 64, wh.ROPE_HALF, [(0, 70), (33, 1), (31, 2), (5, 100)]),
    ("bf16", 64, 1, 8, 128, 48, wh.ROPE_INTERLEAVED, [(0, 200), (64, 64), (63, 2), (100, 1)]),
    ("bf16", 16, 4, 3, 64, 8, wh.ROPE_HALF, [(1, 1), (0, 0), (14, 3), (500, 61)]),
    ("f32", 64, 2, 5, 64, 0, wh.ROPE_HALF, [(10, 129), (0, 63)]),
    ("f16", 16, 1, 1, 128, 120, wh.ROPE_INTERLEAVED, [(7, 2), (8, 8), (1000, 1)]),
]


@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_append(ctx, case):
    kind, page, kh, group, dim, n_rot, layout, steps = case
    rng = np.random.default_rng(len(str(case)) + page)
    st = Step(rng, steps, page, kh, dim, pad=3)
    pool = st.pool(rng)
    # one fused row per token, as a QKV projection leaves it, and a gap behind it
    row = (group + 2) * kh * dim
    qkv, x = typed(ctx, rng, (st.n_tokens, row + 16), kind)
    q, k, v = ((qkv, row + 16, h * dim) for h in (0, group * kh, (group + 1) * kh))
    qx, kx, vx = (x[:, a * dim:b * dim].reshape(st.n_tokens, -1, dim)
                  for a, b in ((0, group * kh), (group * kh, (group + 1) * kh), ((group + 1) * kh, (group + 2) * kh)))
    cos, sin = tables(st.max_kv, n_rot)
    rope, *keep = rope_of(ctx, cos, sin, n_rot, layout) if n_rot else (None,)
    q_out = Array.full(ctx, (st.n_tokens, group * kh, dim), 7.0, kind)
    d = Device(ctx, st, pool)
    d.append(kind, q, k, v, q_out, rope, group * kh)
    got = d.host_pool()
    expect = [a.copy() for a in pool]
    q_ref = ref.append(st, expect, qx, kx, vx, cos.astype(np.float64), sin.astype(np.float64), layout)
    for name, a, b in zip(("k codes", "v codes", "k scales", "v scales"), got, expect):
        assert same_bits(a, b), name
    # rotated in 64 bits, rounded to f32 and to the type: half a step of each
    out = q_out.values()
    used = int(st.cu[-1])
    tol = np.abs(q_ref[:used]) * (ref.EPS[kind] / 2 + 2.0 ** -24) + 1e-7 * (kind == "f16")  # f16 subnormals: 2^-25
    assert np.all(np.abs(out[:used] - q_ref[:used]) <= tol)
    assert np.all(out[used:] == 7.0)  # padding tokens


def test_append_in_steps_equals_its_definition(ctx):
    """Token by token and in chunks: every block's scale only grows, and its codes are those of the definition."""
    rng = np.random.default_rng(11)
    kh, dim, page = 2, 64, 16
    st = Step(rng, [(0, 40), (0, 40)], page, kh, dim)
    pool = st.pool(rng)
    expect = [a.copy() for a in pool]
    d = Device(ctx, st, pool)
    pos = [0, 0]
    # growing values, so that scales change under codes that stay
    for n0, n1 in ((1, 3), (1, 1), (5, 0), (1, 20), (1, 1), (1, 1), (1, 1), (17, 1), (1, 13), (11, 0)):
        part = Step(rng, [(pos[0], n0), (pos[1], n1)], page, kh, dim)
        part.table, part.stride, part.n_pages = st.table, st.stride, st.n_pages
        e = Device(ctx, part, pool)
        e.pool, e.kv = d.pool, d.kv
        size = 1.0 + 0.2 * sum(pos)
        k, kx = typed(ctx, rng, (part.n_tokens, kh, dim), "f32", size)
        v, vx = typed(ctx, rng, (part.n_tokens, kh, dim), "f32", size)
        e.append("f32", None, k, v, None)
        ref.append(part, expect, np.zeros((part.n_tokens, kh, dim)), kx, vx, None, None, 0)
        pos = [pos[0] + n0, pos[1] + n1]
        for a, b in zip(e.host_pool(), expect):
            assert same_bits(a, b), (pos, n0, n1)


def test_append_ties_zeros_and_values_that_are_not_numbers(ctx):
    rng = np.random.default_rng(5)
    kh, dim, page = 1, 64, 16
    st = Step(rng, [(3, 6), (0, 4), (2, 5)], page, kh, dim)
    pool = st.pool(rng)
    pool[2][:] = np.float32(2.0)  # a scale that new values meet in halves
    pool[3][:] = np.float32(0.5)
    k = rng.integers(-400, 400, (15, kh, dim)).astype(np.float32) / 2 * 2
    k[:6] = rng.integers(-253, 254, (6, kh, dim))  # quotients k + 1/2
    v = (rng.integers(-127, 128, (15, kh, dim)) * 0.25).astype(np.float32)
    v[:6, 0, 0] = 127.0  # the scale doubles: odd codes are ties
    k[6:10] = 0.0        # an empty block: scale 0, codes 0
    v[6:10] = np.nan
    k[10, 0, :4] = [np.nan, np.inf, -np.inf, 1e-30]
    v[11, 0, :6] = [np.inf, -np.inf, np.nan, -0.0, 3e38, -3.4028234e38]
    v[12, 0, :] = 1e-45
    expect = [a.copy() for a in pool]
    ref.append(st, expect, np.zeros((15, kh, dim)), k.astype(np.float64), v.astype(np.float64), None, None, 0)
    d = Device(ctx, st, pool)
    d.append("f32", None, Array(ctx, k), Array(ctx, v), None)
    for name, a, b in zip(("k codes", "v codes", "k scales", "v scales"), d.host_pool(), expect):
        assert same_bits(a, b), name
    assert expect[2][st.table[1, 0], 0] == 0 and not expect[0][st.table[1, 0], 0, :4].any()


def test_append_queries_in_place_and_none(ctx):
    rng = np.random.default_rng(6)
    st = Step(rng, [(5, 9), (20, 1)], 16, 2, 64)
    pool = st.pool(rng)
    cos, sin = tables(st.max_kv, 64)
    rope, *keep = rope_of(ctx, cos, sin, 64, wh.ROPE_HALF)
    q, qx = typed(ctx, rng, (10, 4, 64), "f32")
    k, kx = typed(ctx, rng, (10, 2, 64), "f32")
    a, b = Device(ctx, st, pool), Device(ctx, st, pool)
    out = Array.full(ctx, q.shape, 0.0, "f32")
    a.append("f32", q, k, k, out, rope)
    b.append("f32", None, k, k, None, rope)
    assert all(same_bits(x, y) for x, y in zip(a.host_pool(), b.host_pool()))
    b.append("f32", q, k, k, q, rope)
    assert np.array_equal(q.host(), out.host())


def test_append_and_read_skip_what_has_no_place(ctx):
    """Tokens at negative positions, lengths out of their bounds, pages out of the pool."""
    rng = np.random.default_rng(7)
    kh, dim, page = 2, 64, 16
    st = Step(rng, [(10, 8), (0, 6), (4, 5), (20, 20), (0, 3)], page, kh, dim)
    pool = st.pool(rng)
    q, qx = typed(ctx, rng, (st.n_tokens, kh, dim), "f32")
    k, kx = typed(ctx, rng, (st.n_tokens, kh, dim), "f32")
    v, vx = typed(ctx, rng, (st.n_tokens, kh, dim), "f32")
    good = st.table.copy()
    # sequence 1 holds 4 of its 6 tokens, 2 is longer than the bound, 4 has a negative length
    st.kv_len[1], st.kv_len[2], st.kv_len[4] = 4, st.max_kv + 1, -1
    st.table[3, 1] = st.n_pages  # past the pool
    st.table[0, 1] = -1
    d = Device(ctx, st, pool)
    q_out = Array.full(ctx, (st.n_tokens, kh, dim), 7.0, "f32")
    d.append("f32", q, k, v, q_out)
    got = d.host_pool()
    # the same of what has a place: sequence 0's first page, 1's four, 3's first and last page
    expect = [a.copy() for a in pool]
    for s, lo, hi in ((0, 0, 16), (1, 0, 4), (3, 32, 40)):
        start = int(st.kv_len[s] - (st.cu[s + 1] - st.cu[s]))
        for h in range(kh):
            for x, c, sc, turn in ((kx, 0, 2, False), (vx, 1, 3, True)):
                page_id, first = good[s, lo // page], max(start - lo, 0)
                rows = x[st.cu[s] + max(lo, start) - start:st.cu[s] + hi - start, h]
                codes = expect[c][page_id, h].T if turn else expect[c][page_id, h]
                expect[sc][page_id, h] = ref.append_block(rows, codes, first, expect[sc][page_id, h])
    for a, b in zip(got, expect):
        assert same_bits(a, b)
    out = q_out.host()
    live = np.zeros(st.n_tokens, bool)
    live[st.cu[0]:st.cu[1]] = live[st.cu[3]:st.cu[4]] = True
    live[st.cu[1] + 2:st.cu[2]] = True
    assert np.array_equal(out[live], qx[live].astype(np.float32)) and np.all(out[~live] == 7.0)
    ko, vo = (Array.full(ctx, (st.n_tokens, kh, dim), 7.0, "f32") for _ in range(2))
    d.read("f32", ko, vo)
    ko, vo = ko.host(), vo.host()
    assert np.all(ko[~live] == 7.0) and np.all(vo[~live] == 7.0)
    lost = np.zeros(st.n_tokens, bool)
    lost[st.cu[0] + 6:st.cu[1]] = True                # sequence 0's positions 16, 17
    lost[st.cu[3]:st.cu[3] + 12] = True               # sequence 3's positions 20 .. 31
    assert np.isnan(ko[lost]).all() and np.isnan(vo[lost]).all()
    assert np.isfinite(ko[live & ~lost]).all()


# ---------------------------------------------------------------------------
# read back
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind,page,kh,dim,steps", [
    ("f32", 16, 5, 128, [(0, 40), (33, 1), (5, 0), (16, 16)]), ("f16", 32, 2, 64, [(1, 1), (30, 5), (0, 64)]),
    ("bf16", 64, 3, 128, [(0, 130), (62, 3)])])
def test_read(ctx, kind, page, kh, dim, steps):
    rng = np.random.default_rng(page)
    st = Step(rng, steps, page, kh, dim, pad=2)
    pool = st.pool(rng)
    d = Device(ctx, st, pool)
    # rows further apart than their values
    row = kh * dim + 24
    k, v = (Array.full(ctx, (st.n_tokens, row), 7.0, kind) for _ in range(2))
    d.read(kind, (k, row, 0), (v, row, 0))
    for got, which in ((k, 0), (v, 1)):
        want = np.full((st.n_tokens, row), to_kind(7.0, kind))
        for s, (c, n) in enumerate(steps):
            for h in range(kh):
                x = ref.values(st, pool, s, c + n, h)[which][c:]
                want[st.cu[s]:st.cu[s + 1], h * dim:(h + 1) * dim] = to_kind(x, kind)
        assert same_bits(got.host(), want)
    only = Array.full(ctx, (st.n_tokens, row), 7.0, kind)
    d.read(kind, None, (only, row, 0))
    assert same_bits(only.host(), v.host())


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

# type, page, kv heads, group, dim, steps
ATTENTIONS = [
    ("f32", 16, 1, 1, 128, [(0, 1)]),
    ("f32", 16, 5, 4, 128, [(1023, 1)]),
    ("f32", 16, 5, 4, 128, [(0, 1), (63, 1), (64, 1), (300, 1), (15, 1), (0, 0), (255, 1), (256, 1)]),
    ("bf16", 64, 2, 4, 128, [(700, 1), (3, 1), (127, 1)]),
    ("f16", 32, 3, 1, 64, [(100, 1), (31, 1), (32, 1), (500, 2)]),
    ("f32", 32, 2, 3, 64, [(10, 7), (0, 5), (90, 1)]),
    ("bf16", 16, 1, 16, 128, [(40, 1), (333, 2)]),
    ("f32", 16, 1, 40, 128, [(40, 1), (333, 3)]),
    ("f32", 64, 2, 4, 128, [(120, 9), (0, 33), (64, 1)]),
    ("f16", 16, 2, 4, 128, [(0, 150)]),
    ("f32", 32, 1, 4, 128, [(0, 131), (200, 65)]),
    ("bf16", 64, 2, 2, 64, [(0, 200), (70, 1), (0, 64)]),
    ("bf16", 16, 1, 8, 128, [(513, 40), (0, 17)]),
]


def attention_case(ctx, kind, st, pool, rng, heads, size=2.0, scale=None):
    scale = st.dim ** -0.5 if scale is None else scale
    q, qx = typed(ctx, rng, (st.n_tokens, heads, st.dim), kind, size)
    out = Array.full(ctx, (st.n_tokens, heads, st.dim), 7.0, kind)
    lse = Array.full(ctx, (st.n_tokens, heads), 7.0, "f32")
    d = Device(ctx, st, pool)
    d.attend(kind, q, out, lse, scale)
    return d, q, qx, out, lse, scale


def assert_attention(st, pool, kind, qx, out, lse, scale):
    o, z, tol, tol_z = ref.attention(st, pool, qx, scale, kind)
    used = int(st.cu[-1])
    got, got_z = out.values(), lse.values()
    empty = np.isinf(z[:used])
    assert np.array_equal(empty, np.isinf(got_z[:used]) & (got_z[:used] < 0))
    assert np.all(got[:used][empty] == 0)
    err = np.abs(got[:used] - o[:used])
    assert np.all(err <= tol[:used]), (err - tol[:used]).max()
    f = ~empty
    assert np.all(np.abs(got_z[:used][f] - z[:used][f]) <= tol_z[:used][f])
    assert np.all(got[used:] == 7.0) and np.all(got_z[used:] == 7.0)


@pytest.mark.parametrize("case", ATTENTIONS, ids=str)
def test_attention(ctx, case):
    kind, page, kh, group, dim, steps = case
    rng = np.random.default_rng(len(str(case)) + dim)
    st = Step(rng, steps, page, kh, dim, pad=2)
    pool = st.pool(rng)
    _, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, kh * group)
    assert_attention(st, pool, kind, qx, out, lse, scale)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_long(ctx, kind):
    """Many splits of one sequence, next to short ones."""
    rng = np.random.default_rng(3)
    st = Step(rng, [(20000, 1), (5, 1)], 64, 1, 128)
    pool = st.pool(rng)
    _, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, 4)
    assert_attention(st, pool, kind, qx, out, lse, scale)


@pytest.mark.parametrize("group", [4, 20])
def test_attention_rows_without_positions(ctx, group):
    rng = np.random.default_rng(4)
    st = Step(rng, [(0, 6), (0, 3), (300, 2)], 16, 1, 64)
    pool = st.pool(rng)
    st.kv_len[:2] = [4, 0]  # two rows of the first are empty, all of the second
    _, _, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, group)
    assert_attention(st, pool, "f32", qx, out, lse, scale)
    assert np.isinf(lse.host()[[0, 1, 6, 7, 8]]).all()


@pytest.mark.parametrize("steps", [[(40, 1), (100, 1), (60, 1), (33, 1), (9, 1)], [(40, 60), (0, 100), (60, 1), (33, 2), (9, 50)]],
                         ids=["decode", "mixed"])
def test_attention_of_bad_pages_and_lengths_is_nan(ctx, steps):
    rng = np.random.default_rng(8)
    st = Step(rng, steps, 16, 2, 128)
    pool = st.pool(rng)
    st.table[0, 1] = st.n_pages          # a page past the pool
    st.table[1, 3] = -5
    st.kv_len[2], st.kv_len[3] = st.max_kv + 1, -1
    _, _, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 8)
    got, z = out.host(), lse.host()
    for s, (c, n) in enumerate(steps):
        pos = np.arange(c, c + n)
        bad = pos >= 16 if s == 0 else pos >= 48 if s == 1 else np.full(n, s < 4)
        rows, rz = got[st.cu[s]:st.cu[s + 1]], z[st.cu[s]:st.cu[s + 1]]
        assert np.isnan(rows[bad]).all() and np.isnan(rz[bad]).all()
        assert np.isfinite(rows[~bad]).all() and np.isfinite(rz[~bad]).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_attention_over_scales_far_apart(ctx, kind):
    """Blocks of zeros, of tiny and of huge values: none takes another's precision."""
    rng = np.random.default_rng(9)
    st = Step(rng, [(500, 1), (300, 40)], 16, 2, 128)
    pool = st.pool(rng)
    vs, ks = pool[3], pool[2]
    for s in range(2):
        pages = st.table[s, :-(-st.kv_len[s] // 16)]
        vs[pages] *= 2.0 ** rng.integers(-20, 1, (len(pages), 2)).astype(np.float32)
        vs[pages[::5]] = 0.0
        ks[pages[1::7]] = 0.0
    if kind == "f32":
        vs[st.table[0, 3]] = 1e-38
        vs[st.table[1, 2]] = 1e-30
    _, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, 8)
    assert_attention(st, pool, kind, qx, out, lse, scale)


def test_attention_first_block_tiny_then_normal(ctx):
    rng = np.random.default_rng(10)
    st = Step(rng, [(300, 1)], 16, 1, 128)
    pool = st.pool(rng)
    pool[3][st.table[0, 0]] = 1e-37
    _, _, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 4)
    assert_attention(st, pool, "f32", qx, out, lse, scale)


@pytest.mark.parametrize("size,scale", [(1e-20, 1e18), (1e15, 1e-16), (2.0, 0.0), (2.0, -0.09)])
def test_attention_query_sizes_and_scales(ctx, size, scale):
    rng = np.random.default_rng(12)
    st = Step(rng, [(130, 1), (20, 9)], 16, 2, 64)
    pool = st.pool(rng)
    _, _, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 4, size, scale)
    assert_attention(st, pool, "f32", qx, out, lse, scale)


def test_attention_strides_alias_and_no_lse(ctx):
    rng = np.random.default_rng(13)
    st = Step(rng, [(130, 1), (20, 60), (0, 3)], 16, 2, 128)
    pool = st.pool(rng)
    d, q, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 8)
    row = 8 * 128 + 40
    wide = np.full((st.n_tokens, row), np.float32(7.0))
    wide[:, :1024] = q.host().reshape(-1, 1024)
    wide = Array(ctx, wide, "f32")
    d.attend("f32", (wide, row, 0), (wide, row, 0), None, scale, heads=8)  # out over q
    got = wide.host()
    assert np.array_equal(got[:, :1024], out.host().reshape(-1, 1024)) and np.all(got[:, 1024:] == 7.0)


def test_attention_reads_past_4_gib(ctx):
    """Pages beyond byte 2^32 of the pools."""
    rng = np.random.default_rng(14)
    kh, dim, page, far = 5, 128, 64, 110000  # 4.5e9 bytes of codes for K and for V
    st = Step(rng, [(200, 1), (70, 30)], page, kh, dim, spare=0)
    small = st.pool(rng)
    elems = [int(np.prod(x.shape[1:])) * x.itemsize for x in small]
    pool = [ctx.alloc((far + st.n_pages) * n) for n in elems]
    for x, y, n in zip(pool, small, elems):
        ctx.check(wh.lib.wm_memcpy_h2d(ctx.h, x.ptr + far * n, y.ctypes.data, y.nbytes))
    q, qx = typed(ctx, rng, (st.n_tokens, 20, dim), "f32", 2.0)
    k, kx = typed(ctx, rng, (st.n_tokens, kh, dim), "f32")
    d = Device(ctx, st, small)
    d.table.put(np.where(st.table >= 0, st.table + far, st.table))
    d.kv = wh.PagedKV(*[x.ptr for x in pool], far + st.n_pages, page, kh, dim)
    q_out, out, ko = (Array.full(ctx, x.shape, 7.0, "f32") for x in (q, q, k))
    lse = Array.full(ctx, (st.n_tokens, 20), 7.0, "f32")
    d.append("f32", q, k, k, q_out)
    d.attend("f32", q, out, lse, dim ** -0.5)
    d.read("f32", ko, None)
    ref.append(st, small, qx, kx, kx, None, None, 0)
    for x, y, n in zip(pool, small, elems):
        got = np.empty_like(y)
        ctx.check(wh.lib.wm_memcpy_d2h(ctx.h, got.ctypes.data, x.ptr + far * n, got.nbytes))
        assert same_bits(got, y)
    assert_attention(st, small, "f32", qx, out, lse, dim ** -0.5)
    want = np.concatenate([np.stack([ref.values(st, small, s, c + n, h)[0][c:] for h in range(kh)], 1)
                           for s, (c, n) in enumerate(st.steps)])
    assert np.array_equal(ko.host(), want.astype(np.float32))
    for x in pool:
        x.free()


# ---------------------------------------------------------------------------
# together, as a server uses them
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_prompt_then_decode(ctx, kind):
    """Prompts appended and attended to, then eight decode steps: every step's output and the cache."""
    rng = np.random.default_rng(15)
    kh, group, dim, page = 2, 4, 64, 16
    whole = Step(rng, [(0, 60), (0, 31), (0, 9)], page, kh, dim)
    pool = whole.pool(rng)
    expect = [a.copy() for a in pool]
    cos, sin = tables(whole.max_kv, dim)
    rope, *keep = rope_of(ctx, cos, sin, dim, wh.ROPE_HALF)
    shared = None
    pos = [0, 0, 0]
    for new in [(52, 23, 1)] + [(1, 1, 1)] * 8:
        st = Step(rng, list(zip(pos, new)), page, kh, dim)
        st.table, st.stride, st.n_pages = whole.table, whole.stride, whole.n_pages
        d = Device(ctx, st, pool)
        if shared is None:
            shared = d
        d.pool, d.kv = shared.pool, shared.kv
        q, qx = typed(ctx, rng, (st.n_tokens, kh * group, dim), kind, 2.0)
        k, kx = typed(ctx, rng, (st.n_tokens, kh, dim), kind)
        v, vx = typed(ctx, rng, (st.n_tokens, kh, dim), kind)
        q_rot, out = (Array.full(ctx, q.shape, 7.0, kind) for _ in range(2))
        lse = Array.full(ctx, (st.n_tokens, kh * group), 7.0, "f32")
        wh.paged_batch_check(d.kv, d.b, st.cu, st.kv_len, st.table)
        d.append(kind, q, k, v, q_rot, rope)
        d.attend(kind, q_rot, out, lse, dim ** -0.5)
        got = d.host_pool()
        ref.append(st, expect, qx, kx, vx, cos.astype(np.float64), sin.astype(np.float64), wh.ROPE_HALF)
        for a, b in zip(got, expect):
            assert same_bits(a, b)
        assert_attention(st, expect, kind, q_rot.values(), out, lse, dim ** -0.5)
        pos = [p + n for p, n in zip(pos, new)]


def test_captured_step_follows_lengths_and_pages(ctx):
    """One graph of append and attention, replayed for steps whose lengths, pages and values change,
    with eager calls in between; two graphs with workspaces of their own on two streams."""
    rng = np.random.default_rng(16)
    kh, group, dim, page, bound = 2, 4, 128, 16, 640
    other = wh.Context(0)

    def make(c, seed):
        r = np.random.default_rng(seed)
        st = Step(r, [(500, 1), (77, 1), (3, 1)], page, kh, dim, extra_stride=8)
        st.max_kv = bound
        pool = st.pool(r)
        d = Device(c, st, pool)
        d.x = {n: typed(c, r, (3, h, dim), "f32")[0] for n, h in (("q", kh * group), ("k", kh), ("v", kh))}
        d.q_rot, d.out = (Array.full(c, d.x["q"].shape, 7.0, "f32") for _ in range(2))
        d.lse = Array.full(c, (3, kh * group), 7.0, "f32")
        d.ws = Array(c, np.zeros(max(1, wh.paged_attention_workspace(d.kv, d.b, kh * group)), np.uint8))
        cos, sin = tables(bound, dim)
        d.rope, *d.tab = rope_of(c, cos, sin, dim, wh.ROPE_HALF)
        d.host_cos = cos.astype(np.float64), sin.astype(np.float64)
        d.mirror = [a.copy() for a in pool]
        return d

    def step(d):
        d.append("f32", d.x["q"], d.x["k"], d.x["v"], d.q_rot, d.rope)
        d.attend("f32", d.q_rot, d.out, d.lse, dim ** -0.5, d.ws)

    def check(d):
        st = d.st
        x = {n: t.values() for n, t in d.x.items()}
        ref.append(st, d.mirror, x["q"], x["k"], x["v"], *d.host_cos, wh.ROPE_HALF)
        for a, b in zip(d.host_pool(), d.mirror):
            assert same_bits(a, b)
        assert_attention(st, d.mirror, "f32", d.q_rot.values(), d.out, d.lse, dim ** -0.5)

    both = [make(ctx, 1), make(other, 2)]
    graphs = [Graph(d.ctx, lambda d=d: step(d)) for d in both]
    for turn in range(4):
        for d in both:
            st = d.st
            st.kv_len += np.array([1, 5, 0], np.int32) if turn else 0
            need = [-(-int(n) // page) for n in st.kv_len]
            for s_, u in enumerate(need):  # pages for positions that grew past the last
                for lp in range(u):
                    if st.table[s_, lp] < 0:
                        free = sorted(set(range(st.n_pages)) - set(st.table[st.table >= 0].tolist()))
                        st.table[s_, lp] = free[0]
                        for i in (2, 3):
                            d.mirror[i][free[0]] = 0.01
                            d.pool[i].put(d.mirror[i])
            d.len.put(st.kv_len)
            d.table.put(st.table)
            for t in d.x.values():
                t.put(rng.standard_normal(t.shape).astype(np.float32))
        for g in graphs:
            g.replay()
        for d in both:
            check(d)
            step(d)  # eager: the same step again leaves the same
            check(d)
    for g in graphs:
        g.close()
    other.close()


def test_two_contexts(ctx):
    rng = np.random.default_rng(17)
    st = Step(rng, [(700, 1), (50, 3)], 32, 2, 64)
    pool = st.pool(rng)
    other = wh.Context(0)
    _, _, qx, out, lse, scale = attention_case(other, "f32", st, pool, rng, 4)
    assert_attention(st, pool, "f32", qx, out, lse, scale)
    other.close()


# ---------------------------------------------------------------------------
# many sequences, splits, and values at the ends of their ranges
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind,n_seqs,new,group", [
    ("f32", 70, [1], 4), ("bf16", 150, [1, 0, 2], 2), ("f32", 130, [1, 0, 17, 9], 2), ("f16", 66, [20, 33], 1)])
def test_attention_of_many_sequences(ctx, kind, n_seqs, new, group):
    """More than the 64 that a wave scans at a time, with and without long ones among them."""
    rng = np.random.default_rng(n_seqs)
    steps = [(int(rng.integers(0, 40)), new[i % len(new)]) for i in range(n_seqs)]
    steps[3], steps[n_seqs - 2] = (700, 1), (300, 1)
    st = Step(rng, steps, 16, 2, 64, pad=1)
    pool = st.pool(rng)
    _, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, 2 * group)
    assert_attention(st, pool, kind, qx, out, lse, scale)


@pytest.mark.parametrize("kind,page,kh,group,dim,steps", [
    ("f32", 16, 1, 4, 64, [(1500, 40), (0, 20), (700, 1), (900, 0)]),
    ("bf16", 64, 2, 1, 128, [(2000, 17), (3, 130)]),
    ("f16", 32, 1, 6, 64, [(1023, 22), (1024, 21), (255, 1), (256, 3)]),
    ("f32", 64, 1, 33, 128, [(600, 1), (10, 4)])])
def test_attention_of_many_rows_in_splits(ctx, kind, page, kh, group, dim, steps):
    """Few row tiles over long contexts: splits that short sequences do not have."""
    rng = np.random.default_rng(page + group)
    st = Step(rng, steps, page, kh, dim, pad=2)
    pool = st.pool(rng)
    d, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, kh * group)
    assert_attention(st, pool, kind, qx, out, lse, scale)
    # a larger bound divides the step otherwise, and takes more workspace
    st.max_kv, st.max_new = 64 * st.stride if page == 64 else page * st.stride, st.n_tokens
    _, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, kh * group)
    assert_attention(st, pool, kind, qx, out, lse, scale)


def test_more_tokens_than_the_bound_is_nan(ctx):
    rng = np.random.default_rng(18)
    st = Step(rng, [(40, 3), (20, 9), (70, 2)], 16, 2, 64)
    pool = st.pool(rng)
    st.max_new = 8  # the second sequence has 9
    d, q, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 4)
    got, z = out.host(), lse.host()
    assert np.isnan(got[3:12]).all() and np.isnan(z[3:12]).all()
    keep = np.r_[0:3, 12:14]
    o, want_z, tol, tol_z = ref.attention(st, pool, qx, scale, "f32")
    assert np.all(np.abs(got[keep] - o[keep]) <= tol[keep]) and np.all(np.abs(z[keep] - want_z[keep]) <= tol_z[keep])
    # its tokens are not appended, nor read
    k, _ = typed(ctx, rng, (st.n_tokens, 2, 64), "f32")
    before = d.host_pool()
    d.append("f32", None, k, k, None)
    after = d.host_pool()
    pages = st.table[1, :2]
    assert all(same_bits(a[pages], b[pages]) for a, b in zip(before, after))
    ko = Array.full(ctx, (st.n_tokens, 2, 64), 7.0, "f32")
    d.read("f32", ko, None)
    assert np.all(ko.host()[3:12] == 7.0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_of_queries_that_are_not_numbers_stays_in_its_rows(ctx, kind):
    rng = np.random.default_rng(19)
    st = Step(rng, [(100, 2), (40, 30)], 16, 1, 64)
    pool = st.pool(rng)
    qx = rng.standard_normal((st.n_tokens, 4, 64)).astype(np.float32)
    bad = np.zeros((st.n_tokens, 4), bool)
    for at, value in (((0, 1), np.nan), ((5, 2), np.nan), ((9, 0), np.inf), ((20, 3), -np.inf)):
        qx[at][7] = value
        bad[at] = True
    q = Array(ctx, to_kind(qx, kind), kind)
    out = Array.full(ctx, q.shape, 7.0, kind)
    lse = Array.full(ctx, (st.n_tokens, 4), 7.0, "f32")
    d = Device(ctx, st, pool)
    d.attend(kind, q, out, lse, 0.125)
    clean = np.where(bad[..., None], 0, q.values())
    o, z, tol, tol_z = ref.attention(st, pool, clean, 0.125, kind)
    got, got_z = out.values(), lse.values()
    assert np.isnan(got[bad]).all()
    assert np.all(np.abs(got - o)[~bad] <= tol[~bad]) and np.all(np.abs(got_z - z)[~bad] <= tol_z[~bad])


@pytest.mark.parametrize("size", [1e-33, 1e-41, 0.0])
def test_attention_of_tiny_queries(ctx, size):
    rng = np.random.default_rng(20)
    st = Step(rng, [(100, 2), (40, 30)], 16, 1, 64)
    pool = st.pool(rng)
    _, _, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 4, size)
    assert_attention(st, pool, "f32", qx, out, lse, scale)


@pytest.mark.parametrize("first,step", [(-100, 40), (-120, 59), (-60, 25), (100, -50), (-100, 100)])
@pytest.mark.parametrize("steps", [[(90, 1)], [(70, 21)]], ids=["few", "many"])
def test_attention_under_scales_that_rise_past_f32(ctx, steps, first, step):
    """Each page's values are 2^step times the last one's, and only the first page's weights count.

    A block's scale that is below 2^-60 of the power of two 2^e at or above the largest of the row's tiles is taken as
    2^(e - 60): its codes, 127 at most, under weights that sum to one then give up to 127 * 2^(e - 60), with 2^e at most
    twice the largest scale.  That is the second tolerance; the sums themselves stay within their range."""
    rng = np.random.default_rng(21)
    st = Step(rng, steps, 16, 1, 128)
    pool = st.pool(rng)
    pages = st.table[0, :6]
    for i, page in enumerate(pages):
        pool[0][page] = 127 if i == 0 else -127
        pool[2][page] = 1 / 64
        pool[3][page] = 2.0 ** min(first + step * i, 118)
    n = st.n_tokens
    qx = (rng.random((n, 4, 128)) + 0.5).astype(np.float32)
    q = Array(ctx, qx, "f32")
    out, lse = Array.full(ctx, q.shape, 7.0, "f32"), Array.full(ctx, (n, 4), 7.0, "f32")
    d = Device(ctx, st, pool)
    d.attend("f32", q, out, lse, 1.0)
    o, z, tol, tol_z = ref.attention(st, pool, qx.astype(np.float64), 1.0, "f32")
    tol += 127 * 2.0 ** -59 * float(pool[3][pages].max())
    assert np.all(np.abs(out.host() - o) <= tol) and np.all(np.abs(lse.host() - z) <= tol_z)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_captured_ragged_step_follows_its_tokens(ctx, kind):
    """One graph whose sequences take turns being long, short, empty and padded."""
    rng = np.random.default_rng(22)
    kh, group, dim, page, n_tokens, bound = 1, 4, 128, 32, 90, 700
    whole = Step(rng, [(0, 700)] * 4, page, kh, dim)
    pool = whole.pool(rng)
    first = Step(rng, [(0, 1)] * 4, page, kh, dim)
    first.table, first.stride, first.n_pages = whole.table, whole.stride, whole.n_pages
    first.n_tokens, first.max_new, first.max_kv = n_tokens, 80, bound
    d = Device(ctx, first, pool)
    q, k, v = (Array.full(ctx, (n_tokens, h, dim), 0.0, kind) for h in (kh * group, kh, kh))
    q_rot, out = (Array.full(ctx, q.shape, 7.0, kind) for _ in range(2))
    lse = Array.full(ctx, (n_tokens, kh * group), 7.0, "f32")
    ws = Array(ctx, np.zeros(max(1, wh.paged_attention_workspace(d.kv, d.b, kh * group)), np.uint8))

    def call():
        d.append(kind, q, k, v, q_rot)
        d.attend(kind, q_rot, out, lse, 0.09, ws)
    graph = Graph(ctx, call)
    expect = [a.copy() for a in pool]
    for steps in ([(0, 1), (620, 80), (5, 0), (33, 3)], [(699, 1)] * 4, [(0, 0), (0, 0), (690, 10), (0, 79)],
                  [(400, 5), (0, 70), (31, 1), (0, 14)]):
        st = Step(rng, steps, page, kh, dim)
        st.table, st.stride, st.n_pages, st.n_tokens = whole.table, whole.stride, whole.n_pages, n_tokens
        d.cu.put(st.cu)
        d.len.put(st.kv_len)
        x = []
        for a in (q, k, v):
            a.put(to_kind(rng.standard_normal(a.shape), kind))
            x.append(a.values())
        for a in (q_rot, out, lse):
            a.put(np.full(a.shape, to_kind(7.0, a.kind)))
        graph.replay()
        first_out = out.host()
        ref.append(st, expect, *x, None, None, 0)
        assert all(same_bits(a, b) for a, b in zip(d.host_pool(), expect))
        assert_attention(st, expect, kind, q_rot.values(), out, lse, 0.09)
        call()
        assert np.array_equal(out.host(), first_out)
    graph.close()


def test_sequences_share_the_pages_of_a_prefix(ctx):
    """Three sequences read the same first pages, and append into pages of their own."""
    rng = np.random.default_rng(23)
    st = Step(rng, [(70, 1), (66, 20), (64, 2)], 32, 2, 64)
    pool = st.pool(rng)
    st.table[1:, :2] = st.table[0, :2]
    k, kx = typed(ctx, rng, (st.n_tokens, 2, 64), "f32")
    d, q, qx, out, lse, scale = attention_case(ctx, "f32", st, pool, rng, 4)
    assert_attention(st, pool, "f32", qx, out, lse, scale)
    wh.paged_batch_check(d.kv, d.b, st.cu, st.kv_len, st.table)
    d.append("f32", q, k, k, q)
    ref.append(st, pool, qx, kx, kx, None, None, 0)
    assert all(same_bits(a, b) for a, b in zip(d.host_pool(), pool))
    d.attend("f32", q, out, lse, scale)
    assert_attention(st, pool, "f32", qx, out, lse, scale)


# ---------------------------------------------------------------------------
# a row's sums: one decision for all of its lanes
# ---------------------------------------------------------------------------

def under_a_dominating_key(st, rng, tile, later):
    """Zeros of a scale of 0 in the first page, whose fifth key alone scores 100 bits; then tiles of `tile` positions
    with rising value scales: the first one's other keys score 0, `later` (bits, value scale) are those of the next
    tiles, and all behind them score 0 under the first tile's value scale."""
    kc, vc, ks, vs = pool = st.pool(rng)
    ln2 = np.log(2.0)
    kc[:] = 0
    for s in range(len(st.steps)):
        for lp in range(-(-int(st.kv_len[s]) // st.page)):
            page, i = st.table[s, lp], lp * st.page // tile
            ks[page], vs[page] = 1.0, 2.0 ** -3
            if 0 < i <= len(later):
                bits, vs[page] = later[i - 1]
                ks[page] = bits * ln2 / 120
                kc[page, :, :, 0] = rng.integers(112, 125, (st.kh, st.page))
        first = st.table[s, 0]
        kc[first, :, 4, 0], ks[first], vs[first] = 120, 100 * ln2 / 120, 0.0
    return pool


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("kernel", ["few", "many"])
def test_attention_of_a_dominating_key_without_values(ctx, kernel, kind):
    """The fifth key's lane holds a sum that the row's other lanes do not when the value scales rise."""
    rng = np.random.default_rng(24)
    if kernel == "few":
        # 17 rounds of 256 positions of 64 heads: more than 1024 rounds, so that a wave has several tiles
        st, tile, group = Step(rng, [(4200, 1)], 16, 64, 64), 256, 1
    else:
        st, tile, group = Step(rng, [(200, 20)], 16, 2, 64), 64, 4
    pool = under_a_dominating_key(st, rng, tile, [(103, 0.5), (102, 2.0)])
    q = np.zeros((st.n_tokens, st.kh * group, 64), np.float32)
    q[..., 0] = 1.0
    q = Array(ctx, to_kind(q, kind), kind)
    out, lse = Array.full(ctx, q.shape, 7.0, kind), Array.full(ctx, q.shape[:2], 7.0, "f32")
    Device(ctx, st, pool).attend(kind, q, out, lse, 1.0)
    assert_attention(st, pool, kind, q.values(), out, lse, 1.0)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_attention_does_not_depend_on_scales_behind_its_rows(ctx, kind, group):
    """Value scales of a tile's later pages, far above those that a row attends to (rows of the kernel for few and for
    many): within the tolerance of the row's own values, and bit for bit what other scales there leave."""
    rng = np.random.default_rng(25)
    st = Step(rng, [(8, 16), (40, 60)] if group > 1 else [(8, 16), (5, 9)], 16, 1, 64)
    pool = st.pool(rng)
    q, qx = typed(ctx, rng, (st.n_tokens, group, 64), kind, 2.0)
    first = {}
    for step in (100, 70, 1, 0, -30):
        for s in range(2):
            for i, page in enumerate(st.table[s, :-(-int(st.kv_len[s]) // 16)]):
                pool[3][page] = np.float32(1.3) * np.float32(2.0) ** (-100 if i == 0 else min(-100 + step * i, 100))
        out, lse = Array.full(ctx, q.shape, 7.0, kind), Array.full(ctx, q.shape[:2], 7.0, "f32")
        Device(ctx, st, pool).attend(kind, q, out, lse, 0.125)
        o, z, tol, tol_z = ref.attention(st, pool, qx, 0.125, kind)
        # rows that attend to the first page only
        for t in [t for s in range(2) for t in range(st.cu[s], st.cu[s + 1]) if t - st.cu[s] + st.steps[s][0] < 16]:
            assert np.all(np.abs(out.values()[t] - o[t]) <= tol[t]), (step, t)
            # (1e-37 of the tolerance is no more than 2^-22 of these values)
            assert np.abs(o[t]).max() > 2.0 ** -100
            assert np.all(np.abs(lse.values()[t] - z[t]) <= tol_z[t])
            assert same_bits(out.host()[t], first.setdefault(t, out.host()[t])), (step, t)


@pytest.mark.parametrize("cu", [[0, 6, 14], [0, 6, 1 << 30], [3, 6, 10], [-2, 6, 10], [0, -1, 4], [0, 6, 5]],
                         ids=["past", "far-past", "not-from-0", "before-0", "negative", "falls"])
def test_sequences_whose_tokens_break_their_bounds(ctx, cu):
    """Token offsets past the packed arrays, not from 0, negative, falling: such a sequence is not appended nor read, the
    rows of the packed arrays that it has are NaN, and the others are as they are without it."""
    rng = np.random.default_rng(26)
    kh, dim, page = 2, 64, 16
    st = Step(rng, [(0, 6), (16, 4)], page, kh, dim)
    st.max_new = 8
    pool = st.pool(rng)
    st.cu = np.array(cu, np.int32)
    bad = [s for s in range(2) if not 0 <= cu[s] <= cu[s + 1] <= st.n_tokens or (s == 0 and cu[0])]
    good = [s for s in range(2) if s not in bad]
    q, qx = typed(ctx, rng, (st.n_tokens, 4, dim), "f32")
    k, kx = typed(ctx, rng, (st.n_tokens, kh, dim), "f32")
    q_out, out = (Array.full(ctx, q.shape, 7.0, "f32") for _ in range(2))
    ko, vo = (Array.full(ctx, k.shape, 7.0, "f32") for _ in range(2))
    lse = Array.full(ctx, q.shape[:2], 7.0, "f32")
    d = Device(ctx, st, pool)
    with pytest.raises(wh.WillametteError):
        wh.paged_batch_check(d.kv, d.b, st.cu, st.kv_len, st.table)
    d.append("f32", q, k, k, q_out)
    d.read("f32", ko, vo)
    d.attend("f32", q, out, lse, 0.125)
    for a, b in zip(d.host_pool(), pool):
        for s in bad:
            own = st.table[s][st.table[s] >= 0]
            assert same_bits(a[own], b[own])
    # every row: of a good sequence, of a bad one, or of none
    owner = np.full(st.n_tokens, -1)
    for s in range(2):
        owner[max(cu[s], 0):max(cu[s + 1], 0)] = s
    for t, s in enumerate(owner):
        if s in good:
            assert np.array_equal(q_out.host()[t], qx[t].astype(np.float32)) and np.isfinite(ko.host()[t]).all()
            assert np.isfinite(out.host()[t]).all() and np.isfinite(lse.host()[t]).all()
        else:
            assert np.all(q_out.host()[t] == 7.0) and np.all(ko.host()[t] == 7.0) and np.all(vo.host()[t] == 7.0)
            if s in bad:
                assert np.isnan(out.host()[t]).all() and np.isnan(lse.host()[t]).all()
            else:
                assert np.all(out.host()[t] == 7.0) and np.all(lse.host()[t] == 7.0)


@pytest.mark.parametrize("kind,group,pad", [("f32", 4, 0), ("bf16", 20, 0), ("f32", 4, 700)])
def test_attention_in_the_workspace_of_a_larger_step(ctx, kind, group, pad):
    """One workspace, sized for the largest step, serves smaller ones: fewer tokens have more splits.  Padding tokens,
    which no sequence has, take no part in that."""
    rng = np.random.default_rng(27)
    big = Step(rng, [(1500, 300), (900, 200), (100, 30)], 32, 1, 64, pad=pad)
    pool = big.pool(rng)
    kv = wh.PagedKV(0, 0, 0, 0, big.n_pages, 32, 1, 64)
    b = wh.PagedBatch(0, 0, 0, 3, big.stride, big.n_tokens, big.max_new, big.max_kv)
    size = wh.paged_attention_workspace(kv, b, group)
    for steps in ([(1500, 40), (900, 2), (100, 9)], [(1790, 9)], [(1799, 1), (3, 5)], [(0, 300), (700, 12)]):
        st = Step(rng, steps, 32, 1, 64, pad=pad)
        st.table = np.ascontiguousarray(big.table[:len(steps)])
        st.stride, st.n_pages = big.stride, big.n_pages
        d = Device(ctx, st, pool)
        q, qx = typed(ctx, rng, (st.n_tokens, group, 64), kind, 2.0)
        out, lse = Array.full(ctx, q.shape, 7.0, kind), Array.full(ctx, q.shape[:2], 7.0, "f32")
        # full of NaN, and some behind it that stays as it is
        work = Array.full(ctx, (size // 4 + 1000,), np.nan, "f32")
        ctx.check(wh.lib.wm_paged_attention_dev(ctx.h, d.kv, d.b, wh.DTYPES[kind], q.ptr, group * 64, group, 0.125, out.ptr,
                                                group * 64, lse.ptr, work.ptr, size))
        assert_attention(st, pool, kind, qx, out, lse, 0.125)
        assert np.isnan(work.host()[size // 4:]).all()


# ---------------------------------------------------------------------------
# sequences of few rows in more rounds of 256 positions than workgroups: every
# wave has several tiles, runs end inside a sequence's head and span several
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind,page,kh,group,steps", [
    ("f32", 16, 8, 2, [(20000, 1), (9001, 3), (254, 1), (3000, 8), (0, 1), (255, 1), (256, 1)]),
    ("bf16", 64, 16, 1, [(9000, 16), (0, 0), (255, 1), (8191, 1), (700, 2), (5, 1)])])
def test_attention_of_more_rounds_than_workgroups(ctx, kind, page, kh, group, steps):
    rng = np.random.default_rng(28)
    st = Step(rng, steps, page, kh, 64, pad=1)
    assert kh * sum(-(-(c + n) // 256) for c, n in steps if n) > 1024
    pool = st.pool(rng)
    _, _, qx, out, lse, scale = attention_case(ctx, kind, st, pool, rng, kh * group)
    assert_attention(st, pool, kind, qx, out, lse, scale)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("step", [12, -12, 40])
def test_attention_of_rounds_under_rising_scales(ctx, kind, step):
    """Round i of 256 positions has values of 2^(step i) under scores of -step i bits: each round that is kept counts as
    much as the others, at the ordinary tolerance.  (Falling scales stay within 2^-60 of the largest for five rounds, and
    the keys behind them are out of reach.)"""
    rng = np.random.default_rng(29)
    st = Step(rng, [(1279, 1)] * 5, 16, 48, 64)
    kc, vc, ks, vs = pool = st.pool(rng)
    kc[:], ks[:] = 0, 1.0
    for s in range(5):
        for lp in range(80):
            page, i = st.table[s, lp], lp // 16
            kc[page, :, :, 0] = rng.integers(112, 125, (48, 16)) * -np.sign(step)
            ks[page], vs[page] = abs(step) * i * np.log(2.0) / 120, 2.0 ** (step * i - 60)
    q = np.zeros((5, 48, 64), np.float32)
    q[..., 0] = 1.0
    q = Array(ctx, to_kind(q, kind), kind)
    out, lse = Array.full(ctx, q.shape, 7.0, kind), Array.full(ctx, q.shape[:2], 7.0, "f32")
    Device(ctx, st, pool).attend(kind, q, out, lse, 1.0)
    assert_attention(st, pool, kind, q.values(), out, lse, 1.0)


def weight_steps(st, pool, heads):
    """What the steps of small weights can add to an output, beside the 22 bits that the tolerance counts.

    A weight w, relative to a largest one of 2^7 or more, is two f16 terms: h, cut to 11 bits, and w - h.  Below 2^-14
    f16 has steps of 2^-24, so rounding either is off by up to 2^-25, together 2^-24, or 2^-31 of the largest.  A weight
    holds its block's value scale: the largest is at most the row's largest scale, as softmax weights are at most 1, and
    the output's error at most 2^-31 of that times the sum of the codes' sizes."""
    tol = np.zeros((st.n_tokens, heads, st.dim))
    for s in range(len(st.steps)):
        pages = st.table[s, :-(-int(st.kv_len[s]) // st.page)]
        for h in range(heads):
            hk = h // (heads // st.kh)
            codes = np.abs(pool[1][pages, hk].astype(np.int64)).sum((0, 2)) if len(pages) else 0
            tol[st.cu[s]:st.cu[s + 1], h] = 2.0 ** -31 * codes * (pool[3][pages, hk].max() if len(pages) else 0)
    return tol


def test_many_sequences_next_to_a_long_bound(ctx):
    """520 sequences of few tokens in a step whose bound is 8192 each: more blocks and joined rows than one launch counts,
    though hardly any exist."""
    rng = np.random.default_rng(30)
    kh, group, dim, bound = 8, 4, 64, 8192
    steps = [(int(rng.integers(0, 40)), 1) for _ in range(520)]
    steps[3], steps[517], steps[519] = (300, 150), (500, 30), (900, 1)
    st = Step(rng, steps, 16, kh, dim, extra_stride=bound // 16)
    st.n_tokens, st.max_new, st.max_kv = bound, bound, bound
    pool = st.pool(rng)
    expect = [a.copy() for a in pool]
    used = int(st.cu[-1])
    q, qx = typed(ctx, rng, (bound, kh * group, dim), "f32", 2.0)
    k, kx = typed(ctx, rng, (bound, kh, dim), "f32")
    q_out, out = (Array.full(ctx, q.shape, 7.0, "f32") for _ in range(2))
    ko = Array.full(ctx, k.shape, 7.0, "f32")
    lse = Array.full(ctx, q.shape[:2], 7.0, "f32")
    d = Device(ctx, st, pool)
    d.append("f32", q, k, k, q_out)
    d.read("f32", ko, None)
    d.attend("f32", q, out, lse, 0.125)
    ref.append(st, expect, qx, kx, kx, None, None, 0)
    assert all(same_bits(a, b) for a, b in zip(d.host_pool(), expect))
    assert np.array_equal(q_out.host()[:used], q.host()[:used]) and np.all(q_out.host()[used:] == 7.0)
    got = ko.host()
    assert np.all(got[used:] == 7.0)
    for s in (0, 3, 300, 517, 519):
        for h in (0, 7):
            want = ref.values(st, expect, s, int(st.kv_len[s]), h)[0][steps[s][0]:]
            assert np.array_equal(got[st.cu[s]:st.cu[s + 1], h], want.astype(np.float32))
    o, z, tol, tol_z = ref.attention(st, expect, qx, 0.125, "f32")
    tol += weight_steps(st, expect, kh * group)
    assert np.all(np.abs(out.host()[:used] - o[:used]) <= tol[:used])
    assert np.all(np.abs(lse.host()[:used] - z[:used]) <= tol_z[:used])
    assert np.all(out.host()[used:] == 7.0) and np.all(lse.host()[used:] == 7.0)


@pytest.mark.parametrize("page", [16, 64])
def test_appended_in_parts_stays_near_its_values(ctx, page):
    """The same keys and values appended whole, in chunks and one at a time: other codes, as a block's earlier codes are
    rounded again whenever its scale grows, but the same scales, and near the values.

    A code is rounded once when it is stored, by half a step, and once for each later growth of its block's scale, by half
    a step of the scale then, which is no larger than the last: (1 + growths) / 2 steps of the last scale."""
    rng = np.random.default_rng(31)
    kh, dim, n = 2, 64, 150
    whole = Step(rng, [(0, n)], page, kh, dim)
    pool = whole.pool(rng)
    k, kx = typed(ctx, rng, (n, kh, dim), "f32")
    pages = whole.table[0, :-(-n // page)]
    codes = {}
    for name, cuts in (("whole", [n]), ("chunks", [7, 20, 21, 64, 90, n]), ("single", list(range(1, n + 1)))):
        d = Device(ctx, whole, pool)
        growths, before = np.zeros((n, kh, 2), int), None
        at = 0
        for cut in cuts:
            st = Step(rng, [(at, cut - at)], page, kh, dim)
            st.table, st.stride, st.n_pages = whole.table, whole.stride, whole.n_pages
            e = Device(ctx, st, pool)
            e.pool, e.kv = d.pool, d.kv
            part = (k, kh * dim, at * kh * dim)
            e.append("f32", None, part, part, None)
            scales = [x[pages] for x in e.host_pool()[2:]]
            if before is not None:
                for i in range(2):
                    for p in range(at):
                        growths[p, :, i] += scales[i][p // page] > before[i][p // page]
            before, at = scales, cut
        got = d.host_pool()
        codes[name] = got
        for h in range(kh):
            for i, x in enumerate(ref.values(whole, got, 0, n, h)):
                step = np.array([got[2 + i][whole.table[0, p // page], h] for p in range(n)], np.float64)
                tol = step * (1 + growths[:, h, i]) / 2 * (1 + 1e-12)
                assert np.all(np.abs(x - kx[:, h]) <= tol[:, None]), name
        assert growths.any() == (name != "whole")
    for name in ("chunks", "single"):
        assert all(same_bits(codes[name][i][pages], codes["whole"][i][pages]) for i in (2, 3))
        assert not same_bits(codes[name][0][pages], codes["whole"][0][pages])
