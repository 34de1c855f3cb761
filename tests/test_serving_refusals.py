"""The serving operators without a GPU: bad arguments are refused on the host
before anything is launched, sizes are what the header says, and host tensors
are refused by the wrappers."""
import pytest
import torch

from nativebit_amd import _lib, ops
from tests.conftest import gpu_available

P = 0x100000   # aligned, never dereferenced
F32, BF16 = _lib.NB_F32, _lib.NB_BF16
EINVAL, EUNSUP, EALIGN = _lib.NB_EINVAL, _lib.NB_EUNSUPPORTED, _lib.NB_EALIGN


def call(name, **kw):
    return getattr(_lib.load(), name)(*kw.values())


def plan(**kw):
    a = dict(table=P, stride=4, lens=P + 16, new=P + 32, free=P + 48, state=P + 64, R=3, width=4,
             n_blocks=20, n_tokens=5, slots=P + 80, positions=P + 96, chunks=P + 112,
             lens_out=P + 128, state_out=P + 144, stream=None)
    return call("nb_kv_plan", **{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(R=0), EINVAL), (dict(width=0), EINVAL), (dict(n_blocks=0), EINVAL),
    (dict(R=4097), EUNSUP), (dict(width=1 << 25, stride=1 << 25), EUNSUP),
    (dict(n_blocks=1 << 25), EUNSUP), (dict(stride=3), EINVAL), (dict(n_tokens=-1), EINVAL),
    (dict(R=4096, n_tokens=1 << 20), EUNSUP), (dict(table=None), EINVAL), (dict(lens=None), EINVAL),
    (dict(new=None), EINVAL), (dict(free=None), EINVAL), (dict(state=None), EINVAL),
    (dict(slots=None), EINVAL), (dict(chunks=None), EINVAL), (dict(positions=None), EINVAL),
    (dict(lens_out=None), EINVAL), (dict(state_out=None), EINVAL),
    (dict(lens_out=P + 16), EINVAL), (dict(state_out=P + 64), EINVAL), (dict(lens_out=P + 32), EINVAL),
    (dict(slots=P + 81), EALIGN), (dict(lens=P + 17), EALIGN), (dict(table=P + 2), EALIGN),
])
def test_plan_refuses(kw, status):
    assert plan(**kw) == status and _lib.last_error()


def release(**kw):
    a = dict(table=P, stride=4, lens=P, finished=P, free=P, state=P, R=3, width=4, n_blocks=20,
             stream=None)
    return call("nb_kv_release", **{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(R=0), EINVAL), (dict(R=4097), EUNSUP), (dict(stride=1), EINVAL), (dict(finished=None), EINVAL),
    (dict(lens=None), EINVAL), (dict(free=None), EINVAL), (dict(state=P + 1), EALIGN),
    (dict(R=4096, width=1 << 20, stride=1 << 20), EUNSUP),
])
def test_release_refuses(kw, status):
    assert release(**kw) == status


def append(**kw):
    a = dict(qkv=P, qkv_dtype=F32, ld=4 * 3 * 32, slots=P, positions=P, chunks=P, n_chunks=2, cos=P,
             sin=P, n_pos=10, k=P, v=P, ks=P, vs=P, n_blocks=5, q=P + (1 << 20), q_dtype=F32, ld_q=8 * 32,
             n_tokens=7, n_head=8, n_kv=2, D=32, stream=None)
    return call("nb_kv8_append", **{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(n_head=9), EINVAL), (dict(n_kv=0), EINVAL), (dict(n_head=0), EINVAL), (dict(D=24), EUNSUP),
    (dict(D=272), EUNSUP), (dict(D=0), EUNSUP), (dict(n_blocks=0), EINVAL), (dict(n_tokens=-1), EINVAL),
    (dict(ld=12 * 32 - 1), EINVAL), (dict(ld_q=255), EINVAL), (dict(qkv_dtype=2), EINVAL),
    (dict(q_dtype=7), EINVAL), (dict(k=P + 8), EALIGN), (dict(ks=P + 1), EALIGN), (dict(k=None), EINVAL),
    (dict(qkv=None), EINVAL), (dict(slots=None), EINVAL), (dict(chunks=None), EINVAL),
    (dict(n_chunks=-1), EINVAL), (dict(n_pos=-1), EINVAL), (dict(qkv=P + 2), EALIGN),
    (dict(cos=None), EINVAL), (dict(sin=P + 2), EALIGN), (dict(n_chunks=1 << 24), EUNSUP),
    (dict(n_head=40000, n_kv=40000, ld=1 << 30, ld_q=1 << 30), EUNSUP),
])
def test_append_refuses(kw, status):
    assert append(**kw) == status


def read(**kw):
    a = dict(slots=P, n=7, k=P, v=P, ks=P, vs=P, n_blocks=5, n_kv=2, D=32, keys=P, values=P,
             dtype=F32, stream=None)
    return call("nb_kv8_read", **{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(n=-1), EINVAL), (dict(n=1 << 30), EUNSUP), (dict(D=8), EUNSUP), (dict(n_kv=0), EINVAL),
    (dict(keys=None), EINVAL), (dict(values=P + 2), EALIGN), (dict(dtype=2), EINVAL),
    (dict(slots=None), EINVAL), (dict(slots=P + 2), EALIGN), (dict(v=None), EINVAL),
])
def test_read_refuses(kw, status):
    assert read(**kw) == status


def attention(**kw):
    a = dict(q=P, q_dtype=F32, ld_q=256, chunks=P, n_chunks=2, lens=P, table=P, stride=4, R=3,
             width=4, k=P, v=P, ks=P, vs=P, n_blocks=5, out=P + (1 << 20), out_dtype=BF16, ld_out=256, n_tokens=7,
             n_head=8, n_kv=2, D=32, softcap=0.0, window=0, slopes=None, prefix=None, ws=None,
             ws_bytes=0, stream=None)
    return call("nb_kv8_attention", **{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(n_head=7), EINVAL), (dict(D=260), EUNSUP), (dict(R=0), EINVAL), (dict(width=5), EINVAL),
    (dict(ld_q=255), EINVAL), (dict(ld_out=255), EINVAL), (dict(q_dtype=2), EINVAL),
    (dict(out_dtype=2), EINVAL), (dict(out=None), EINVAL), (dict(q=P + 2), EALIGN),
    (dict(chunks=None), EINVAL), (dict(lens=None), EINVAL), (dict(softcap=-1.0), EINVAL),
    (dict(softcap=float("nan")), EINVAL), (dict(softcap=float("inf")), EINVAL), (dict(softcap=1e-25), EINVAL),
    (dict(window=-1), EINVAL), (dict(slopes=P + 2), EALIGN), (dict(prefix=P + 1), EALIGN),
    (dict(n_chunks=1 << 23), EUNSUP), (dict(table=None), EINVAL),
    # few chunks over a long cache need a workspace
    (dict(width=4000, stride=4000), EINVAL),
    (dict(width=4000, stride=4000, ws=P, ws_bytes=100), EINVAL),
    (dict(width=4000, stride=4000, ws=P + 8, ws_bytes=1 << 30), EALIGN),
])
def test_attention_refuses(kw, status):
    assert attention(**kw) == status


def logits(**kw):
    a = dict(logits=P, dtype=F32, ld=100, rows=3, V=100, history=P, ld_history=9, max_history=9,
             lens=P, prompt=P, rep=P, freq=P, pres=P, ids=P, bias=P, ld_bias=4, n_bias=4, mask=P,
             ld_mask=4, out=P + 4096, ld_out=100, tokens=P, ws=P, ws_bytes=1 << 20, stream=None)
    return call("nb_logits_rules", **{**a, **kw})


@pytest.mark.parametrize("kw,status", [
    (dict(rows=-1), EINVAL), (dict(V=0), EINVAL), (dict(rows=65536), EUNSUP), (dict(ld=99), EINVAL),
    (dict(ld_out=99), EINVAL), (dict(dtype=2), EINVAL), (dict(logits=None), EINVAL),
    (dict(out=None), EINVAL), (dict(history=None), EINVAL), (dict(lens=None), EINVAL),
    (dict(history=None, lens=None), EINVAL), (dict(ld_history=8), EINVAL), (dict(max_history=-1), EINVAL),
    (dict(n_bias=-1), EINVAL), (dict(ids=None), EINVAL), (dict(bias=None), EINVAL),
    (dict(ld_bias=3), EINVAL), (dict(ld_mask=3), EINVAL), (dict(mask=P + 2), EALIGN),
    (dict(tokens=P + 2), EALIGN), (dict(V=50257, ld=50257, ld_out=50257, ld_mask=1571, ws_bytes=8), EINVAL),
    (dict(V=50257, ld=50257, ld_out=50257, ld_mask=1571, ws=None), EINVAL),
    (dict(out=P, dtype=BF16), EINVAL), (dict(out=P, ld_out=101), EINVAL),
    (dict(out=P + 4), EINVAL), (dict(out=P + 1196), EINVAL), (dict(out=P - 1196), EINVAL),
])
def test_logits_refuses(kw, status):
    assert logits(**kw) == status


Q_ROW, QKV_ROW = 8 * 32 * 4, 12 * 32 * 4   # bytes


@pytest.mark.parametrize("f,kw,fits", [
    # in place; the same memory in another type or stride, or moved
    (append, dict(q=P, ld_q=384), True), (append, dict(q=P), False), (append, dict(q=P, n_tokens=1), True),
    (append, dict(q=P, ld_q=384, q_dtype=BF16), False), (append, dict(q=P + 4, ld_q=384), False),
    # in front, behind, one element into it
    (append, dict(q=P - 7 * Q_ROW), True), (append, dict(q=P - 7 * Q_ROW + 4), False),
    (append, dict(q=P + 7 * QKV_ROW), True), (append, dict(q=P + 7 * QKV_ROW - 4), False),
    # columns beside it in rows of 640 and 639
    (append, dict(ld=640, ld_q=640, q=P + QKV_ROW), True),
    (append, dict(ld=640, ld_q=640, q=P - Q_ROW), True),
    (append, dict(ld=639, ld_q=639, q=P + QKV_ROW), False),
    (attention, dict(out=P, out_dtype=F32), True), (attention, dict(out=P), False),
    (attention, dict(out=P, out_dtype=F32, ld_out=512), False),
    (attention, dict(out=P - 7 * 512), True), (attention, dict(out=P - 7 * 512 + 2), False),
    (attention, dict(out=P + 7 * 1024), True), (attention, dict(out=P + 7 * 1024 - 2), False),
    (attention, dict(out=P + 1024, ld_q=512, ld_out=512, out_dtype=F32), True),
    (attention, dict(out=P + 1020, ld_q=512, ld_out=512, out_dtype=F32), False),
    (logits, dict(out=P), True), (logits, dict(out=P + 400, ld=200, ld_out=200), True),
    (logits, dict(out=P + 396, ld=200, ld_out=200), False),
])
def test_outputs_over_inputs(f, kw, fits):
    if fits and gpu_available():
        pytest.skip("a GPU is there: the call would run")
    assert f(**kw) == (_lib.NB_ENODEV if fits else EINVAL)


def test_nothing_to_do_is_no_error():
    assert append(n_tokens=0) == 0 and read(n=0) == 0 and attention(n_tokens=0) == 0
    assert append(n_chunks=0) == 0 and attention(n_chunks=0) == 0 and logits(rows=0) == 0


def test_valid_calls_need_a_device():
    if gpu_available():
        pytest.skip("a GPU is there")
    for f in (plan, release, append, read, attention, logits):
        assert f() == _lib.NB_ENODEV


def test_chunk_bound():
    """The bound holds for the worst split of rows over blocks: each request's
    first row the last of a block, so that n rows touch (n - 2) / 64 + 2 blocks."""
    lib = _lib.load()
    for R in (1, 2, 5, 64, 4096):
        for n in (0, 1, 2, 3, 63, 64, 65, 66, 67, 129, 130, 1000, 5000, 70000):
            bound = lib.nb_kv_plan_chunks(n, R)
            assert bound == ops.kv_plan_chunks(n, R) <= n
            for active in {min(R, n), min(R, n // 2), 1} - {0}:
                if not n:
                    continue
                share = [n // active + (i < n % active) for i in range(active)]
                assert sum((s - 2) // 64 + 2 if s > 1 else 1 for s in share) <= bound


def test_workspaces():
    lib = _lib.load()
    assert lib.nb_kv8_attention_ws_bytes(0, 0, 4, 8, 2, 32) == 0
    assert lib.nb_kv8_attention_ws_bytes(5, 5, 8, 20, 20, 128) == 0          # short caches
    nbytes = lib.nb_kv8_attention_ws_bytes(6, 6, 626, 32, 8, 128)            # few long ones
    assert nbytes > 0 and nbytes % (6 * 32 * 130 * 4) == 0
    assert lib.nb_logits_rules_ws_bytes(3, 1000) == 0
    assert lib.nb_logits_rules_ws_bytes(300, 50257) == 300 * 25 * 8
    assert lib.nb_logits_rules_ws_bytes(1, 50257) == 50 * 8


def test_wrappers_refuse_host_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv_plan(t, i, i, i, i, 2)
    with pytest.raises(ValueError):
        ops.kv_release(t, i, i, i, i)
    k, s = torch.zeros(1, 1, 64, 16, dtype=torch.int8), torch.zeros(1, 1)
    p = ops.KVPlan(i, i, t, i, i)
    with pytest.raises(ValueError):
        ops.kv8_read(i, k, k, s, s)
    with pytest.raises(ValueError):
        ops.kv8_append(torch.zeros(2, 48), p, s, s, k, k, s, s, 1)
    with pytest.raises(ValueError):
        ops.kv8_attention(torch.zeros(2, 16), p, t, k, k, s, s)
    with pytest.raises(ValueError):
        ops.logits_rules(torch.zeros(2, 5))
