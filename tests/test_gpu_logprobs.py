"""nr_token_logprobs against 64 bits: statistics, ties, masked, NaN and infinite logits."""
import math

import pytest

torch = pytest.importorskip("torch")

from kv8_util import DTYPES, stream  # noqa: E402
from nitrorag_b200._lib import lib  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for gpu tests")


def call(x, targets, k, want_entropy=True, expect=0):
    """x [M, V], any row stride."""
    M, V = x.shape
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[x.dtype]
    tl = torch.full((M,), 77.0, device="cuda") if targets is not None else None
    en = torch.full((M,), 77.0, device="cuda") if want_entropy else None
    tp = torch.full((M, k), 77.0, device="cuda") if k else None
    ids = torch.full((M, k), -7, dtype=torch.int32, device="cuda") if k else None
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    rc = lib().nr_token_logprobs(x.data_ptr(), code, x.stride(0), M, V, ptr(targets), k, ptr(tl), ptr(en), ptr(tp), ptr(ids),
                                 stream())
    assert rc == expect
    return tl, en, tp, ids


def ranked(x, k):
    """Ids of the k largest, equal ones by id, NaN behind -inf."""
    y = torch.where(x.isnan(), torch.full_like(x, -math.inf), x.float())
    order = torch.sort(y, dim=-1, descending=True, stable=True).indices
    if bool(x.isnan().any()):
        nan = torch.gather(x.isnan(), 1, order)
        order = torch.gather(order, 1, torch.sort(nan.int(), dim=-1, stable=True).indices)
    return order[:, :k].int()


def check(x, k, seed=0):
    M, V = x.shape
    targets = torch.randint(0, V, (M,), device="cuda", dtype=torch.int32, generator=torch.Generator(device="cuda").manual_seed(seed))
    tl, en, tp, ids = call(x, targets, k)
    lp = torch.log_softmax(x.double(), -1)
    p = lp.exp()
    # y = x - max and its exp to fp32 (2^-22 relative each), sums of V positive terms (well under 2^-18 with
    # partial sums per thread); log of the sum carries that as an absolute error; the entropy a weighted mean of |y|
    ls = 2.0 ** -18
    want = lp.gather(1, targets.long()[:, None])[:, 0]
    fine = want.isfinite()
    assert torch.equal(tl[~fine].double().nan_to_num(0.5), want[~fine].nan_to_num(0.5))
    assert bool(((tl[fine].double() - want[fine]).abs() <= ls + 2.0 ** -23 * want[fine].abs()).all())
    y = torch.where(p > 0, (x.double() - x.double().amax(-1, keepdim=True)).abs(), torch.zeros_like(p))
    h = -torch.xlogy(p, p).sum(-1)
    room = ls + 2.0 ** -18 * (p * y).sum(-1)
    fine = h.isfinite()
    assert torch.equal(en.isnan(), h.isnan())
    assert bool(((en.double() - h).abs() <= room)[fine].all()), (en, h)
    if k:
        assert torch.equal(ids, ranked(x, k))
        want = lp.gather(1, ids.long())
        fine = want.isfinite()
        assert torch.equal(tp[~fine].double().nan_to_num(0.5), want[~fine].nan_to_num(0.5))
        assert bool(((tp[fine].double() - want[fine]).abs() <= ls + 2.0 ** -23 * want[fine].abs()).all())


def logits(M, V, dtype, seed, pad=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (spread * torch.randn((M, V + pad), generator=g, device="cuda")).to(DTYPES[dtype][1])
    return x[:, :V]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,V,k,pad", [(1, 1, 1, 0), (3, 2, 2, 1), (5, 31, 31, 0), (2, 33, 32, 3), (7, 1000, 5, 0), (4, 1001, 20, 0),
                                       (64, 32000, 5, 0), (1, 32000, 0, 0), (1, 128256, 32, 0), (2, 50001, 7, 5), (300, 4099, 3, 0),
                                       (1, 300007, 32, 1), (2, 1000003, 4, 0)])
def test_logprobs(dtype, M, V, k, pad):
    check(logits(M, V, dtype, V + k, pad), k)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [257, 32000, 128256])
def test_order_of_ties(dtype, V):
    """Few distinct values, one value throughout, +-0, the largest at the ends, rising and falling rows."""
    dt = DTYPES[dtype][1]
    g = torch.Generator(device="cuda").manual_seed(V)
    few = torch.randint(0, 3, (1, V), generator=g, device="cuda").float()
    rise = torch.arange(V, device="cuda").float()[None] * (100.0 / V)
    ends = torch.zeros((1, V), device="cuda")
    ends[0, -1] = ends[0, 0] = 3.0
    zero = torch.zeros((1, V), device="cuda")
    zero[0, ::2] = -0.0
    x = torch.cat([few, torch.full((1, V), -2.5, device="cuda"), zero, ends, rise, rise.flip(1)]).to(dt)
    for k in (1, 8, 32):
        check(x, k)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [40, 5000, 128256])
def test_masked_and_non_finite(dtype, V):
    """Forbidden words (-inf and the type's lowest value), all but one or all of a row forbidden, NaN, +inf."""
    dt = DTYPES[dtype][1]
    x = logits(9, V, dtype, 1).clone()
    low = torch.finfo(dt).min
    x[0, torch.rand(V, device="cuda") < 0.7] = -math.inf
    x[1, torch.rand(V, device="cuda") < 0.7] = low
    x[2] = -math.inf
    x[2, V // 2] = 1.0
    x[3] = low
    x[3, V - 1] = 1.0
    x[4] = -math.inf
    x[5] = low
    x[6, V // 3] = math.nan
    x[7, V // 3] = math.inf
    x[8, :V - 2] = math.nan
    for k in (1, 5, 32):
        check(x, k)


def test_targets_and_optional_outputs():
    x = logits(6, 777, "bf16", 3)
    t = torch.tensor([0, 776, 777, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    tl, en, tp, ids = call(x, t, 2)
    assert bool(tl[:2].isfinite().all()) and bool(tl[2:].isnan().all()) and bool(en.isfinite().all())
    only = call(x, t, 0, want_entropy=False)
    assert torch.equal(only[0][:2], tl[:2])
    only = call(x, None, 2, want_entropy=False)
    assert torch.equal(only[2], tp) and torch.equal(only[3], ids)
    assert torch.equal(call(x, None, 0)[1], en)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_any_alignment(dtype):
    """Rows that start at any element, so that no two of them are aligned the same way."""
    base = logits(1, 40000, dtype, 9).reshape(-1)
    for off in (0, 1, 3, 7):
        x = torch.as_strided(base, (11, 3001), (3003, 1), off)
        check(x, 6)


def test_offsets_past_32_bits():
    V = 128256
    M = (1 << 31) // V + 9
    x = torch.zeros((M, V), dtype=torch.bfloat16, device="cuda")
    x[-3:] = logits(3, V, "bf16", 4)
    _, en, tp, ids = call(x, None, 5)
    _, en3, tp3, ids3 = call(x[-3:].clone(), None, 5)
    # few rows are cut among more CTAs than many, so their sums are taken in another order: each side is
    # within 2^-18 + 2^-23 |value| (and the entropy's 2^-18 sum p |y|, under 2^-18 * 10 here) of 64 bits
    assert torch.equal(ids[-3:], ids3)
    assert bool(((tp[-3:] - tp3).abs() <= 2 * (2.0 ** -18 + 2.0 ** -23 * tp3.abs())).all())
    assert bool(((en[-3:] - en3).abs() <= 2 * 11 * 2.0 ** -18).all())


def test_graph_replay():
    x = logits(5, 32000, "f32", 5).clone()
    want = call(x, None, 4)
    out = [torch.zeros_like(want[1]), torch.zeros_like(want[2]), torch.zeros_like(want[3])]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc = lib().nr_token_logprobs(x.data_ptr(), 0, x.stride(0), 5, 32000, None, 4, None, out[0].data_ptr(), out[1].data_ptr(),
                                     out[2].data_ptr(), stream())
    assert rc == 0
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[1:]))
        x.copy_(logits(5, 32000, "f32", 6))
        want = call(x, None, 4)
