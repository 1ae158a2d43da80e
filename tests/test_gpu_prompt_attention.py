"""nr_prompt_attention against 64-bit causal attention, sequence by sequence."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from kv8_util import DTYPES, assert_within, attend, bound, i32, stream  # noqa: E402
from nitrorag_b200._lib import lib  # noqa: E402

pytestmark = pytest.mark.gpu

# weights enter the second product in the inputs' type; exp2 to 2^-13
P_ROUND = {"bf16": 2.0 ** -8 + 2.0 ** -13, "f16": 2.0 ** -11 + 2.0 ** -13}


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for gpu tests")


def call(q, k, v, out, cu_q, cu_k, B, H, KV, hd, err=None, Tq=None, Tk=None, expect=0):
    code = DTYPES["bf16" if q.dtype == torch.bfloat16 else "f16"][0]
    rc = lib().nr_prompt_attention(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                   out.data_ptr(), out.stride(0), code, cu_q.data_ptr(),
                                   None if cu_k is None else cu_k.data_ptr(), B, len(q) if Tq is None else Tq,
                                   len(k) if Tk is None else Tk, H, KV, hd, None if err is None else err.data_ptr(), stream())
    assert rc == expect


def reference(q, k, v, lens_q, lens_k, H, KV, hd, at_q=0, at_k=0):
    n = len(q)
    out, pv = (torch.zeros((n, H, hd), dtype=torch.float64, device="cuda") for _ in range(2))
    size, small = torch.zeros((n, H), dtype=torch.float64, device="cuda"), torch.zeros_like(out)
    for a, b in zip(lens_q, lens_k):
        seen = torch.arange(b, device="cuda")[None] <= torch.arange(a, device="cuda")[:, None] + (b - a)
        for h in range(H if a else 0):
            j = h // (H // KV)
            cut = lambda x, lo, m, i: x[lo:lo + m, i * hd:(i + 1) * hd].double()  # noqa: E731
            out[at_q:at_q + a, h], pv[at_q:at_q + a, h], size[at_q:at_q + a, h] = attend(
                cut(q, at_q, a, h), cut(k, at_k, b, j), cut(v, at_k, b, j), seen)
            small[at_q:at_q + a, h] = seen.double() @ cut(v, at_k, b, j).abs()
        at_q += a
        at_k += b
    return out, (pv, size), small


def check(dtype, lens_q, lens_k, H, KV, hd, seed=0, pad=0, scale=1.0, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[dtype][1]
    nq, nk = sum(lens_q) + pad, sum(lens_k) + pad
    if packed:  # one wide row; queries and keys are the same tokens
        rows = torch.randn((nq, (H + 2 * KV) * hd + 8), generator=g, device="cuda").to(dt)
        q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:(H + 2 * KV) * hd]
    else:
        q = (scale * torch.randn((nq, H * hd), generator=g, device="cuda")).to(dt)
        k, v = (torch.randn((nk, KV * hd), generator=g, device="cuda").to(dt) for _ in range(2))
    if pad:  # rows behind the last sequence hold anything
        for x in (q, k, v):
            x[-pad:] = float("nan")
    out = torch.full((nq, H * hd + 8), 5.0, dtype=dt, device="cuda")
    cu_q, cu_k = (i32([0] + np.cumsum(x).tolist()) for x in (lens_q, lens_k))
    err = i32([0])
    call(q, k, v, out[:, :H * hd], cu_q, None if packed else cu_k, len(lens_q), H, KV, hd, err)
    want, scores, small = reference(q, k, v, lens_q, lens_k, H, KV, hd)
    n = sum(lens_q)
    assert int(err) == 0
    got = out[:, :H * hd].reshape(-1, H, hd)
    assert_within(got[:n], want[:n], bound(dtype, want, *scores, P_ROUND[dtype], small)[:n], "prompt")
    assert bool((out[n:] == 5).all()) and bool((out[:, H * hd:] == 5).all())
    again = torch.full_like(out, 5.0)
    call(q, k, v, again[:, :H * hd], cu_q, None if packed else cu_k, len(lens_q), H, KV, hd, err)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd,H,KV", [(64, 2, 2), (128, 4, 2), (64, 3, 1), (128, 5, 5), (64, 8, 1)])
@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255, 256, 257], [1, 0, 17, 300, 0, 64, 5], [600, 3, 385]])
def test_prompts(dtype, hd, H, KV, lens):
    check(dtype, lens, lens, H, KV, hd, seed=sum(lens) + H, pad=sum(lens) % 3, packed=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd,H,KV", [(64, 4, 2), (128, 2, 1)])
@pytest.mark.parametrize("lens_q,lens_k", [([1, 1, 1], [1, 500, 128]), ([5, 130, 0, 64], [5, 700, 3, 65]), ([40, 300], [0, 129]),
                                           ([200, 1], [72, 0]), ([129], [128]), ([16, 17], [1000, 1023])])
def test_chunks(dtype, hd, H, KV, lens_q, lens_k):
    """Queries that are the last tokens of longer keys; queries with fewer keys than themselves (their first
    rows see nothing and give zeros); sequences without keys."""
    check(dtype, lens_q, lens_k, H, KV, hd, seed=sum(lens_k), pad=2)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [1e-3, 20.0])
def test_flat_and_peaked(dtype, scale):
    check(dtype, [513, 100], [513, 100], 4, 2, 128, seed=3, scale=scale)
    check(dtype, [513, 100], [513, 100], 2, 2, 64, seed=4, scale=scale)


def test_rising_scores():
    """The maximum grows by hundreds from block to block: the running output is rescaled each time."""
    n, hd = 700, 128
    dt = torch.bfloat16
    u = torch.randn(hd, device="cuda")
    u /= u.norm()
    q = (40 * u + 0.1 * torch.randn((n, hd), device="cuda")).to(dt)
    k = (torch.arange(n, device="cuda")[:, None] * 0.25 * u + 0.5 * torch.randn((n, hd), device="cuda")).to(dt)
    v = torch.randn((n, hd), device="cuda").to(dt)
    for kk in (k, k.flip(0).contiguous()):
        out = torch.empty_like(q)
        call(q, kk, v, out, i32([0, n]), None, 1, 1, 1, hd)
        want, scores, _ = reference(q, kk, v, [n], [n], 1, 1, hd)
        assert_within(out.reshape(n, 1, hd), want, bound("bf16", want, *scores, P_ROUND["bf16"]), "rising")


@pytest.mark.parametrize("hd", [64, 128])
def test_neighbours_hold_anything(hd):
    """A sequence of NaN and infinities between two others, and its rows' neighbours within one tile."""
    lens, H, KV = [37, 50, 90], 2, 1
    n = sum(lens)
    rows = torch.randn((n, (H + 2 * KV) * hd), device="cuda").to(torch.bfloat16)
    clean = rows.clone()
    rows[37:87] = float("nan")
    rows[50:60] = float("inf")
    cu = i32([0, 37, 87, n])
    outs = []
    for r in (clean, rows):
        out = torch.zeros((n, H * hd), dtype=r.dtype, device="cuda")
        call(r[:, :H * hd], r[:, H * hd:(H + KV) * hd], r[:, (H + KV) * hd:], out, cu, None, 3, H, KV, hd)
        outs.append(out)
    assert torch.equal(outs[0][:37], outs[1][:37]) and torch.equal(outs[0][87:], outs[1][87:])


def test_out_of_range_rows_are_skipped_and_flagged():
    H = KV = 2
    hd, n = 64, 300
    q, k, v = (torch.randn((n, H * hd), device="cuda").to(torch.float16) for _ in range(3))
    good = torch.full_like(q, 5.0)
    cu = [0, 100, 180, 300]
    call(q, k, v, good, i32(cu), None, 3, H, KV, hd)
    for bad_q, bad_k, skipped in (([0, 100, 180, 301], cu, [2]), (cu, [0, 100, 180, 301], [2]), (cu, [-1, 100, 180, 300], [0]),
                                  (cu, [0, 100, 90, 300], [1])):
        out, err = torch.full_like(q, 5.0), i32([0])
        call(q, k, v, out, i32(bad_q), i32(bad_k), 3, H, KV, hd, err)
        assert int(err) == 2
        for b in range(3):
            rows = slice(cu[b], cu[b + 1])
            if b in skipped:
                assert bool((out[rows] == 5).all())
            elif bad_k[b:b + 2] == cu[b:b + 2]:
                assert torch.equal(out[rows], good[rows])


def test_graph_and_stream():
    H, KV, hd, n = 4, 2, 128, 333
    rows = torch.randn((n, (H + 2 * KV) * hd), device="cuda").to(torch.bfloat16)
    parts = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:]
    out, want = (torch.zeros((n, H * hd), dtype=rows.dtype, device="cuda") for _ in range(2))
    cu = i32([0, 300, n])
    call(*parts, want, cu, None, 2, H, KV, hd)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(*parts, out, cu, None, 2, H, KV, hd)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    rows.copy_(torch.randn_like(rows))
    call(*parts, want, cu, None, 2, H, KV, hd)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("H,KV", [(4, 2), (5, 5), (1, 1)])
def test_long_among_short(dtype, H, KV):
    """head_dim 128, 32 tokens and less on average, one of the sequences of many key blocks."""
    lens = [1, 0, 3, 7, 2] * 20
    lens[33] = 901
    check(dtype, lens, lens, H, KV, 128, seed=H, pad=3)
    check(dtype, [min(n, 140) for n in lens], lens, H, KV, 128, seed=H + 1)


def test_many_sequences():
    rng = np.random.default_rng(1)
    check("bf16", rng.integers(0, 4, 1024).tolist(), rng.integers(0, 4, 1024).tolist(), 1, 1, 64, seed=5, pad=1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens,H,KV,hd", [([700, 130], 4, 2, 128), ([700, 130], 3, 3, 128), ([5] * 60 + [290], 2, 1, 128),
                                          ([700, 130], 4, 2, 64)])
@pytest.mark.parametrize("level,step", [(-60, 0), (60, 0), (-90, 12), (90, -12), (0, 12)])
def test_weights_of_the_old_maximum_never_stay(dtype, lens, H, KV, hd, level, step):
    """Scores near `level` that move by `step` from one block of 128 keys to the next: the weights taken
    from the maximum so far (0 before the first block) would be infinite or nothing, so that one of
    them left among the new maximum's shows.  Every tiling: two heads, two tiles of a head, one tile."""
    dt = DTYPES[dtype][1]
    g = torch.Generator(device="cuda").manual_seed(hd + H + len(lens))
    n = sum(lens)
    q = (0.05 * torch.randn((n, H, hd), generator=g, device="cuda"))
    k = torch.randn((n, KV, hd), generator=g, device="cuda")
    at = torch.cat([torch.arange(m, device="cuda") for m in lens])
    q[:, :, 0] = 8.0  # the score's level, in one dim: 8 k / sqrt(hd)
    k[:, :, 0] = ((level + step * (at // 128)).float() * hd ** 0.5 / 8.0)[:, None]
    q, k = q.to(dt).reshape(n, -1), k.to(dt).reshape(n, -1)
    v = torch.randn((n, KV * hd), generator=g, device="cuda").to(dt)
    cu = i32([0] + np.cumsum(lens).tolist())
    out = torch.full_like(q, 5.0)
    call(q, k, v, out, cu, None, len(lens), H, KV, hd)
    want, scores, small = reference(q, k, v, lens, lens, H, KV, hd)
    assert_within(out.reshape(n, H, hd), want, bound(dtype, want, *scores, P_ROUND[dtype], small), "prompt")
