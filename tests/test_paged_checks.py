"""CPU checks of the paged cache and token scores: every refusal of a call,
made before the device is touched (on a context without one), and the check
of a step's arrays on host copies."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import willamette_hip as wh
from paged_ref import Step

ROOT = Path(__file__).resolve().parent.parent
GOOD = 1 << 20  # stands for an aligned device address; never read


@pytest.fixture(scope="module")
def hctx(tmp_path_factory):
    so = tmp_path_factory.mktemp("host_ctx") / "host_ctx.so"
    subprocess.run(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17",
                    "-shared", "-fPIC", f"-I{ROOT / 'include'}", f"-I{ROOT / 'project-willamette_amd/csrc'}", "-w",
                    "-o", str(so), str(ROOT / "tests/host_ctx.cpp")], check=True)
    lib = C.CDLL(str(so))
    lib.host_ctx.restype = C.c_void_p
    return lib.host_ctx()


def descriptors(**over):
    kv = dict(k_codes=GOOD, v_codes=GOOD, k_scales=GOOD, v_scales=GOOD, n_pages=8, page_size=16, n_kv_heads=2,
              head_dim=128)
    b = dict(cu_tokens=GOOD, kv_len=GOOD, page_table=GOOD, n_seqs=2, table_stride=4, n_tokens=10, max_new=6,
             max_kv_len=64)
    for k, v in over.items():
        (kv if k in kv else b)[k] = v
    return wh.PagedKV(**kv), wh.PagedBatch(**b)


def append(ctx, kv, b, rope=None, type_=0, q=GOOD, qs=1024, heads=8, k=GOOD, ks=256, v=GOOD, vs=256, o=GOOD, os=1024):
    return wh.lib.wm_paged_kv_append_dev(ctx, kv, b, rope, type_, q, qs, heads, k, ks, v, vs, o, os)


def read(ctx, kv, b, type_=0, k=GOOD, ks=256, v=GOOD, vs=256):
    return wh.lib.wm_paged_kv_read_dev(ctx, kv, b, type_, k, ks, v, vs)


def attend(ctx, kv, b, type_=0, q=GOOD, qs=1024, heads=8, scale=0.1, o=GOOD, os=1024, lse=GOOD, work=GOOD, size=1 << 40):
    return wh.lib.wm_paged_attention_dev(ctx, kv, b, type_, q, qs, heads, scale, o, os, lse, work, size)


CALLS = {"append": append, "read": read, "attend": attend}
ARG, SHAPE, TYPE, NONFINITE, BOUNDS = 6, 2, 1, 3, 13


@pytest.mark.parametrize("call", sorted(CALLS))
@pytest.mark.parametrize("over,status", [
    (dict(k_codes=0), ARG), (dict(v_codes=0), ARG), (dict(k_scales=0), ARG), (dict(v_scales=0), ARG),
    (dict(k_codes=GOOD + 8), ARG), (dict(v_codes=GOOD + 4), ARG), (dict(k_scales=GOOD + 2), ARG),
    (dict(n_pages=0), SHAPE), (dict(n_pages=1 << 31), SHAPE), (dict(page_size=0), SHAPE), (dict(page_size=8), SHAPE),
    (dict(page_size=48), SHAPE), (dict(page_size=128), SHAPE), (dict(head_dim=0), SHAPE), (dict(head_dim=96), SHAPE),
    (dict(head_dim=256), SHAPE), (dict(n_kv_heads=0), SHAPE), (dict(n_kv_heads=65537), SHAPE),
    (dict(cu_tokens=0), ARG), (dict(kv_len=0), ARG), (dict(page_table=0), ARG), (dict(cu_tokens=GOOD + 1), ARG),
    (dict(kv_len=GOOD + 2), ARG), (dict(page_table=GOOD + 3), ARG), (dict(table_stride=3), SHAPE),
    (dict(max_kv_len=65), SHAPE), (dict(max_new=11), SHAPE), (dict(n_tokens=1 << 31), SHAPE),
    (dict(max_kv_len=(1 << 30) + 1, table_stride=1 << 31), SHAPE), (dict(n_seqs=0xFFFFFFFF), SHAPE)])
def test_descriptor_refusals(hctx, call, over, status):
    kv, b = descriptors(**over)
    assert CALLS[call](hctx, kv, b) == status
    assert wh.lib.wm_last_error(hctx)


@pytest.mark.parametrize("call", sorted(CALLS))
def test_null_arguments(hctx, call):
    kv, b = descriptors()
    assert CALLS[call](None, kv, b) == ARG
    assert CALLS[call](hctx, None, b) == ARG
    assert CALLS[call](hctx, kv, None) == ARG
    assert CALLS[call](hctx, kv, b, type_=2) == TYPE
    assert CALLS[call](hctx, kv, b, type_=-1) == TYPE


def test_array_refusals(hctx):
    kv, b = descriptors()
    for bad, status in ((dict(q=None), ARG), (dict(q=GOOD + 4), ARG), (dict(qs=1022), ARG), (dict(qs=1020), SHAPE),
                        (dict(o=None), ARG), (dict(o=GOOD + 8), ARG), (dict(os=1025), ARG), (dict(os=512), SHAPE),
                        (dict(heads=7), SHAPE), (dict(qs=1 << 41), SHAPE)):
        assert append(hctx, kv, b, **bad) == status, bad
        assert attend(hctx, kv, b, **bad) == status, bad
    for bad, status in ((dict(k=GOOD + 4), ARG), (dict(ks=254), ARG), (dict(ks=252), SHAPE), (dict(v=GOOD + 4), ARG),
                        (dict(vs=254), ARG), (dict(vs=128), SHAPE)):
        assert append(hctx, kv, b, **bad) == status, bad
        assert read(hctx, kv, b, **bad) == status, bad
    assert append(hctx, kv, b, k=None) == ARG and append(hctx, kv, b, v=None) == ARG
    # half types: eight elements to 16 bytes
    assert append(hctx, kv, b, type_=30, ks=260) == ARG and attend(hctx, kv, b, type_=1, qs=1028) == ARG
    assert attend(hctx, kv, b, heads=0) == SHAPE
    assert attend(hctx, kv, b, lse=GOOD + 2) == ARG
    for s in (float("nan"), float("inf"), -float("inf")):
        assert attend(hctx, kv, b, scale=s) == NONFINITE


def test_rope_refusals(hctx):
    kv, b = descriptors()
    for args, status in (((0, GOOD, 64, 128, 0), ARG), ((GOOD, 0, 64, 128, 0), ARG), ((GOOD + 4, GOOD, 64, 128, 0), ARG),
                         ((GOOD, GOOD, 63, 128, 0), SHAPE), ((GOOD, GOOD, 64, 12, 0), SHAPE),
                         ((GOOD, GOOD, 64, 136, 0), SHAPE), ((GOOD, GOOD, 64, 128, 2), ARG)):
        assert append(hctx, kv, b, rope=wh.Rope(*args)) == status, args


def test_workspace_refusals(hctx):
    kv, b = descriptors(max_kv_len=4096, table_stride=256, n_pages=1000)
    need = wh.paged_attention_workspace(kv, b, 8)
    assert need > 0
    assert attend(hctx, kv, b, size=need - 1) == ARG
    assert attend(hctx, kv, b, work=None) == ARG
    assert attend(hctx, kv, b, work=GOOD + 8) == ARG
    # nothing to divide by, and no workspace of a call that is refused anyway
    assert wh.paged_attention_workspace(wh.PagedKV(), b, 8) == 0
    assert wh.paged_attention_workspace(kv, b, 7) == 0


def test_nothing_to_do(hctx):
    """No sequences or no tokens: fine without any array, and without a device."""
    for over in (dict(n_seqs=0), dict(n_tokens=0, max_new=0)):
        kv, b = descriptors(**over)
        for call in CALLS.values():
            assert call(hctx, kv, b) == 0
    kv, b = descriptors()
    assert read(hctx, kv, b, k=None, v=None) == 0


def step(seed=0, **kw):
    st = Step(np.random.default_rng(seed), [(20, 3), (0, 33), (15, 1), (7, 0)], 16, 2, 128, **kw)
    kv = wh.PagedKV(0, 0, 0, 0, st.n_pages, 16, 2, 128)
    b = wh.PagedBatch(0, 0, 0, 4, st.stride, st.n_tokens, st.max_new, st.max_kv)
    return st, kv, b


def check(st, kv, b, appends=True):
    try:
        wh.paged_batch_check(kv, b, st.cu, st.kv_len, st.table, appends)
    except wh.WillametteError as e:
        return e.status
    return 0


def test_batch_check_accepts_a_step():
    st, kv, b = step(pad=5)
    assert check(st, kv, b) == 0 and check(st, kv, b, False) == 0
    # entries past a sequence's pages, and of one without tokens, are not looked at
    st.table[3] = 1 << 30
    assert check(st, kv, b) == 0
    # two sequences that share a full page of a common beginning
    st.table[2, 0], st.kv_len[2], st.table[2, 1] = st.table[0, 0], 17, st.table[2, 0]
    assert check(st, kv, b) == 0
    # a sequence longer than its cache
    st.kv_len[1] = 30
    assert check(st, kv, b) == 0


def test_batch_check_refuses():
    def broken(change, appends=True):
        st, kv, b = step()
        change(st, kv, b)
        return check(st, kv, b, appends)

    def put(name, i, x):
        def f(st, kv, b):
            getattr(st, name)[i] = x
        return f
    assert broken(put("cu", 0, 1)) == SHAPE
    assert broken(put("cu", 1, -1)) == SHAPE
    assert broken(put("cu", 2, 2)) == SHAPE      # falls
    assert broken(put("cu", 4, 38)) == SHAPE     # past n_tokens
    assert broken(put("kv_len", 0, -1)) == SHAPE
    assert broken(put("kv_len", 0, 34)) == SHAPE  # past max_kv_len
    for x in (-1, 1 << 30, -(1 << 31)):
        assert broken(put("table", (0, 0), x)) == BOUNDS
        assert broken(put("table", (1, 2), x), False) == BOUNDS
    # a page appended to twice: by two sequences, by one, or read by another
    assert broken(lambda st, kv, b: st.table.__setitem__((2, 0), st.table[1, 0])) == BOUNDS
    assert broken(lambda st, kv, b: st.table.__setitem__((2, 0), st.table[1, 0]), False) == 0
    assert broken(lambda st, kv, b: st.table.__setitem__((1, 1), st.table[1, 0])) == BOUNDS
    assert broken(lambda st, kv, b: st.table.__setitem__((0, 0), st.table[2, 0])) == BOUNDS
    assert broken(lambda st, kv, b: setattr(kv, "page_size", 8)) == SHAPE
    assert broken(lambda st, kv, b: setattr(b, "max_new", 40)) == SHAPE


def scores(ctx, type_=0, x=GOOD, stride=100, rows=3, vocab=100, tok=GOOD, k=5, lp=GOOD, en=GOOD, rk=GOOD, ids=GOOD,
           tlp=GOOD, work=GOOD, size=1 << 40):
    return wh.lib.wm_token_logprobs_dev(ctx, type_, x, stride, rows, vocab, tok, k, lp, en, rk, ids, tlp, work, size)


@pytest.mark.parametrize("bad,status", [
    (dict(type_=7), TYPE), (dict(vocab=0), SHAPE), (dict(vocab=1 << 31), SHAPE), (dict(rows=1 << 31), SHAPE),
    (dict(k=65), SHAPE), (dict(k=5, vocab=4, stride=4), SHAPE), (dict(stride=99), SHAPE), (dict(stride=1 << 41), SHAPE),
    (dict(k=0), ARG), (dict(k=0, ids=None), ARG), (dict(tok=None), ARG), (dict(tok=None, lp=None), ARG),
    (dict(x=None), ARG), (dict(x=GOOD + 2), ARG), (dict(type_=30, x=GOOD + 1), ARG), (dict(tok=GOOD + 2), ARG),
    (dict(lp=GOOD + 1), ARG), (dict(en=GOOD + 1), ARG), (dict(rk=GOOD + 1), ARG), (dict(ids=GOOD + 1), ARG),
    (dict(tlp=GOOD + 1), ARG)], ids=str)
def test_logprobs_refusals(hctx, bad, status):
    assert scores(hctx, **bad) == status
    assert wh.lib.wm_last_error(hctx)


def test_logprobs_null_context_and_no_rows(hctx):
    assert scores(None) == ARG
    assert scores(hctx, rows=0, x=None) == 0
    f = wh.lib.wm_token_logprobs
    assert f(None, None, 1, 5, None, 0, None, None, None, None, None) == ARG
    assert f(hctx, None, 1, 5, None, 0, None, None, None, None, None) == ARG
    assert f(hctx, None, 0, 5, None, 0, None, None, None, None, None) == 0
    x = np.zeros(5, np.float32)
    assert f(hctx, x.ctypes.data_as(C.POINTER(C.c_float)), 1, 5, None, 65, None, None, None, None, None) == SHAPE


def test_workspaces_of_sizes_that_no_call_takes():
    """Sizes whose plan would divide by nothing or leave 32 bits: no workspace, and no fault."""
    for over in (dict(n_seqs=0), dict(n_tokens=0), dict(max_new=0), dict(max_new=0xFFFFFFFF, n_tokens=0xFFFFFFFF),
                 dict(max_kv_len=0xFFFFFFFF), dict(max_new=1 << 31, n_tokens=1 << 31, n_seqs=1 << 31)):
        kv, b = descriptors(**over)
        assert wh.paged_attention_workspace(kv, b, 64) == 0
    for rows, vocab in ((1, 0xFFFFFFFF), (1, 0xFFFFFFFA), (1, 0xFFFFFFF2), (0, 5000), (3, (1 << 30) + 1)):
        assert wh.token_logprobs_workspace(rows, vocab, 5) == 0


def test_attention_refuses_more_workgroups_than_a_launch_has(hctx):
    kv, b = descriptors(n_kv_heads=4096, n_seqs=4096, max_kv_len=1024, table_stride=64, n_tokens=4096, max_new=1)
    assert attend(hctx, kv, b, heads=4096, qs=4096 * 128, os=4096 * 128) == SHAPE
    kv, b = descriptors(n_seqs=1 << 20, n_kv_heads=16, n_tokens=1 << 20, max_new=64)
    assert attend(hctx, kv, b, heads=64, qs=64 * 128, os=64 * 128) == SHAPE


def test_attention_workspace_covers_smaller_steps():
    """The size falls with no bound: what a server allocates for its largest step serves all others."""
    rng = np.random.default_rng(0)
    names = ("n_seqs", "n_tokens", "max_new", "max_kv_len")
    for turn in range(3000):
        most = [int(2 ** x) for x in rng.uniform(0, (8, 14, 12, 15))]
        most[2] = min(most[2], most[1])
        less = [max(1, int(m * rng.choice([1, 1, rng.random(), rng.random() ** 4]))) for m in most]
        less[2] = min(less[2], less[1])
        kvh, group = int(rng.choice([1, 2, 5, 8])), int(rng.choice([1, 4, 8, 33]))
        sizes = []
        for bounds in (most, less):
            kv, b = descriptors(n_kv_heads=kvh, table_stride=1 << 12, **dict(zip(names, bounds)))
            sizes.append(wh.paged_attention_workspace(kv, b, kvh * group))
        assert sizes[1] <= sizes[0], (most, less, kvh, group, sizes)
        assert sizes[0] <= 110_000_000 + 8300 * kvh * most[0]
    # a long prompt, and the chunk of it that a smaller step has
    kv, b = descriptors(n_kv_heads=5, n_seqs=1, n_tokens=8192, max_new=8192, max_kv_len=8192, table_stride=512)
    whole = wh.paged_attention_workspace(kv, b, 20)
    for n in (2048, 512, 100, 10, 1):
        b.n_tokens = b.max_new = n
        assert wh.paged_attention_workspace(kv, b, 20) <= whole


def test_logprobs_workspace_covers_smaller_calls():
    """Few rows are taken in short parts, many in long ones: what serves many serves few."""
    rng = np.random.default_rng(1)
    for turn in range(5000):
        most = [int(2 ** x) for x in rng.uniform(0, (11, 18))] + [int(rng.integers(0, 65))]
        less = [max(1, int(m * rng.choice([1, 1, rng.random()]))) for m in most[:2]] + [int(rng.integers(0, most[2] + 1))]
        assert wh.token_logprobs_workspace(*less) <= wh.token_logprobs_workspace(*most), (most, less)
    for rows in range(1, 700):
        assert wh.token_logprobs_workspace(rows, 128256, 20) <= wh.token_logprobs_workspace(rows + 1, 128256, 20), rows


def test_output_over_its_queries_has_their_stride(hctx):
    """With another stride a row's output would fall on queries that are still to be read."""
    kv, b = descriptors()
    for call in (append, attend):
        assert call(hctx, kv, b, qs=1024, os=1040) == ARG
        assert call(hctx, kv, b, qs=1040, os=1024) == ARG


def test_attention_refuses_a_scale_without_a_base_2_form(hctx):
    """Scores are formed in base 2: scale * log2 e has to be finite too."""
    kv, b = descriptors()
    for s in (2.4e38, -3.4e38):
        assert attend(hctx, kv, b, scale=s) == NONFINITE


def test_logprobs_host_form_refuses_before_it_copies(hctx):
    """Sizes that the device form refuses are refused before anything is allocated or read."""
    x = np.zeros(5, np.float32)
    p = x.ctypes.data_as(C.POINTER(C.c_float))
    f = wh.lib.wm_token_logprobs
    assert f(hctx, p, 1, (1 << 30) + 1, None, 0, None, None, None, None, None) == SHAPE
    assert f(hctx, p, 1 << 31, 5, None, 0, None, None, None, None, None) == SHAPE
    assert f(hctx, p, 1, 5, None, 6, None, None, None, None, None) == SHAPE
    ids = (C.c_int32 * 5)()
    assert f(hctx, p, 1, 5, None, 0, None, None, None, ids, None) == ARG
    lp = (C.c_float * 5)()
    assert f(hctx, p, 1, 5, None, 0, lp, None, None, None, None) == ARG
