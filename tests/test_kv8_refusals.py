"""Argument checks of the 8-bit page, prompt attention and log probability entry points.  A refused
call returns before anything is launched, so these run without a GPU (addresses are never read)."""
import ctypes as C

import pytest

from nitrorag_b200._lib import NrKv8AppendArgs, NrKv8Pool, lib

A = 0x10000  # a 16-byte aligned address that no refused call touches
INVALID = -1


def pool(**kw):
    f = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, n_layers=2, n_kv_heads=2, head_dim=64)
    return NrKv8Pool(**{**f, **kw})


BAD_POOLS = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=A + 8), dict(v=A + 1), dict(n_pages=0),
             dict(n_layers=0), dict(n_kv_heads=0), dict(n_kv_heads=-1), dict(head_dim=96), dict(head_dim=0)]


def append_args(**kw):
    f = dict(q=A, k=A, v=A, q_out=A, k_out=A, q_stride=256, k_stride=128, v_stride=128, q_out_stride=256, k_out_stride=128,
             cu_seqlens=A, start_pos=A, block_tables=A, rope_cos=A, rope_sin=A, dtype=1, B=1, T=1, n_heads=4, max_pages=2,
             layer=0, rope_len=8, rot_dim=64, rope_layout=0)
    return NrKv8AppendArgs(**{**f, **kw})


@pytest.mark.parametrize("kw", BAD_POOLS)
def test_pools(kw):
    p, a = pool(**kw), append_args()
    assert lib().nr_kv8_append(C.byref(p), C.byref(a), None, None) == INVALID
    assert lib().nr_paged_attention_decode_kv8(A, 1, C.byref(p), 0, A, 2, A, 1, 4, A, A, None, None) == INVALID


@pytest.mark.parametrize("kw", [
    dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(cu_seqlens=None), dict(start_pos=None), dict(block_tables=None),
    dict(rope_cos=None), dict(rope_sin=None), dict(rope_cos=A + 4), dict(rope_len=0), dict(dtype=3), dict(dtype=-1), dict(B=0),
    dict(B=1025), dict(T=0), dict(n_heads=0), dict(max_pages=0), dict(layer=2), dict(layer=-1), dict(rot_dim=8), dict(rot_dim=80),
    dict(rot_dim=-16), dict(rope_layout=2), dict(q=A + 2), dict(k=A + 8), dict(v=A + 4), dict(q_out=A + 2), dict(k_out=A + 2),
    dict(q_stride=255), dict(q_stride=248), dict(k_stride=127), dict(k_stride=132), dict(v_stride=0), dict(k_out_stride=64),
    dict(q_out_stride=264), dict(k_out_stride=136),  # in place with another stride
    dict(max_pages=(1 << 26) + 1),  # 2^30 positions
])
def test_append(kw):
    p, a = pool(), append_args(**kw)
    assert lib().nr_kv8_append(C.byref(p), C.byref(a), None, None) == INVALID


def test_append_null_structs():
    p, a = pool(), append_args()
    assert lib().nr_kv8_append(None, C.byref(a), None, None) == INVALID
    assert lib().nr_kv8_append(C.byref(p), None, None, None) == INVALID


DECODE = dict(q=A, dtype=1, layer=0, bt=A, max_pages=2, ctx=A, B=1, n_heads=4, out=A, ws=A)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(bt=None), dict(ctx=None), dict(out=None), dict(ws=None), dict(dtype=3), dict(layer=2), dict(layer=-1),
    dict(max_pages=0), dict(B=0), dict(B=1025), dict(n_heads=0), dict(n_heads=3), dict(n_heads=34), dict(q=A + 2), dict(out=A + 8),
    dict(ws=A + 4), dict(max_pages=(1 << 26) + 1)])
def test_decode(kw):
    p, d = pool(), {**DECODE, **kw}
    assert lib().nr_paged_attention_decode_kv8(d["q"], d["dtype"], C.byref(p), d["layer"], d["bt"], d["max_pages"], d["ctx"],
                                               d["B"], d["n_heads"], d["out"], d["ws"], None, None) == INVALID


def test_decode_workspace_size():
    size = lib().nr_paged_attention_kv8_workspace_size
    assert size(1, 4, 2, 64, 2) > 0
    assert size(1024, 32, 8, 128, 8192) > 0
    for bad in ((0, 4, 2, 64, 2), (1025, 4, 2, 64, 2), (1, 0, 2, 64, 2), (1, 4, 0, 64, 2), (1, 5, 2, 64, 2), (1, 34, 2, 64, 2),
                (1, 4, 2, 65, 2), (1, 4, 2, 64, 0)):
        assert size(*bad) == 0


@pytest.mark.parametrize("H,KV,hd", [(32, 32, 128), (17, 17, 64), (32, 8, 128), (16, 1, 64), (20000, 20000, 64)])
def test_decode_workspace_size_never_falls_with_the_batch(H, KV, hd):
    """One workspace, sized for the largest batch, serves every smaller one: the sizes never fall, and each
    holds the counters, a partial result for each unit of a batch that is cut (up to 16384 items of a
    sequence and kv head are), and the list of units of up to 32 items."""
    group, before = H // KV, 0
    rec = (group * hd + (2 * group + 3) // 4 * 4) * 4
    for b in range(1, 1025):
        size = lib().nr_paged_attention_kv8_workspace_size(b, H, KV, hd, 2048)
        assert size >= before
        before = size
        items = b * KV
        assert size >= 4 * 16384 + ((items + 2 * 148 * 5) * rec if items <= 16384 else 0) + (8 * items if items <= 32 else 0)


PROMPT = dict(q=A, qs=256, k=A, ks=128, v=A, vs=128, out=A, os=256, dtype=1, cu_q=A, cu_k=None, B=1, Tq=8, Tk=8, H=4, KV=2, hd=64)


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(cu_q=None), dict(dtype=0), dict(dtype=3), dict(B=0), dict(B=1025),
    dict(Tq=0), dict(Tk=0), dict(Tk=9), dict(H=0), dict(KV=0), dict(H=5), dict(hd=32), dict(q=A + 2), dict(k=A + 8), dict(v=A + 8),
    dict(out=A + 2), dict(qs=255), dict(qs=260), dict(ks=120), dict(vs=129), dict(os=0)])
def test_prompt(kw):
    d = {**PROMPT, **kw}
    assert lib().nr_prompt_attention(d["q"], d["qs"], d["k"], d["ks"], d["v"], d["vs"], d["out"], d["os"], d["dtype"], d["cu_q"],
                                     d["cu_k"], d["B"], d["Tq"], d["Tk"], d["H"], d["KV"], d["hd"], None, None) == INVALID


SCORE = dict(x=A, dtype=1, ld=100, M=2, V=100, t=A, k=5, tl=A, en=A, tp=A, ids=A)


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(x=A + 1), dict(dtype=3), dict(ld=99), dict(M=0), dict(V=0), dict(k=-1), dict(k=33), dict(V=4), dict(t=None),
    dict(tl=None), dict(tp=None), dict(ids=None), dict(k=0), dict(t=None, tl=None, en=None, k=0, tp=None, ids=None)])
def test_score(kw):
    d = {**SCORE, **kw}
    assert lib().nr_token_logprobs(d["x"], d["dtype"], d["ld"], d["M"], d["V"], d["t"], d["k"], d["tl"], d["en"], d["tp"], d["ids"],
                                   None) == INVALID


def test_every_unit_of_packed_rows_is_covered():
    """The kernels give sequence b the units cu[b]//W + n*b and up; every tile (n = 1) or page (n = 2) of
    a sequence falls on a unit of its own, below T//W + n*B."""
    import random
    rng = random.Random(3)
    for _ in range(300):
        lens = [rng.choice([0, 1, 2, 15, 16, 17, 127, 128, 129, rng.randrange(1000)]) for _ in range(rng.randint(1, 40))]
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        for W, n in ((128, 1), (16, 2)):
            for b, m in enumerate(lens):
                start = rng.randrange(100) if n == 2 else 0
                pieces = (start + m - 1) // W - start // W + 1 if m else 0
                room = cu[b + 1] // W + n * (b + 1) - (cu[b] // W + n * b)
                assert pieces <= room


def test_engine_logprobs_without_gpu():
    from nitrorag_b200 import EngineConfig, NitroEngine, NrError
    eng = NitroEngine(config=EngineConfig(total_blocks=8, device=-1), shape=(64, 128, 2, 2, 2, 100, 64))
    with pytest.raises(NrError, match="NO_DEVICE"):
        eng.last_decode_logprobs(top_k=1)
    f, i = (C.c_float * 8)(), (C.c_int32 * 8)()
    call = lib().nr_decode_last_logprobs
    for args in ((None, -1, None, f, None, None, None), (None, 33, None, f, f, i, None), (None, 0, None, None, None, None, None),
                 (i, 0, None, f, None, None, None), (None, 0, f, f, None, None, None), (None, 1, None, f, None, i, None),
                 (None, 0, None, f, f, i, None)):
        assert call(eng._h, *args) == INVALID
    assert call(None, None, 0, None, f, None, None, None) == INVALID
    eng.close()
