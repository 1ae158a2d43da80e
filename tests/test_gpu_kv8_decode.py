"""nr_paged_attention_decode_kv8 against 64-bit attention over the same codes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from kv8_util import DTYPES, PAGE, Pool, assert_within, attend, bound, decode, i32, tables  # noqa: E402
from nitrorag_b200._lib import lib  # noqa: E402

pytestmark = pytest.mark.gpu

# weights enter the products as fp16 (16-bit types) or as two fp16 halves (fp32)
P_ROUND = {"f32": 2.0 ** -20, "bf16": 2.0 ** -11, "f16": 2.0 ** -11}


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for gpu tests")


def reference(pool, q, table, ctx, layer, pages_ok=None):
    """(out, sum p|v|, size) in 64 bits; page ids outside the pool are absent tokens."""
    B, H, hd = q.shape
    n_pages, _, KV, _ = pool.shape4
    out, pv, size = (torch.zeros(s, dtype=torch.float64, device="cuda") for s in ((B, H, hd), (B, H, hd), (B, H)))
    for b in range(B):
        n = min(max(int(ctx[b]), 0), table.shape[1] * PAGE)
        ids = table[b, :(n + PAGE - 1) // PAGE].long()
        there = (ids >= 0) & (ids < n_pages)
        here = there.repeat_interleave(PAGE)[:n]
        ids = torch.where(there, ids, torch.zeros_like(ids))
        for j in range(KV):
            kk, vv = (getattr(pool, x)[ids, layer, j].view(torch.float8_e4m3fn).double()
                      * getattr(pool, x + "_scale")[ids, layer, j].double()[:, None, None] for x in "kv")
            kk, vv = (t.reshape(-1, hd)[:n][here] for t in (kk, vv))
            g = H // KV
            seen = torch.ones((g, len(kk)), dtype=torch.bool, device="cuda")
            r = attend(q[b, j * g:(j + 1) * g].double(), kk, vv, seen)
            out[b, j * g:(j + 1) * g], pv[b, j * g:(j + 1) * g], size[b, j * g:(j + 1) * g] = r
    return out, pv, size


def check(pool, q, table, ctx, layer, dtype, flag=0, **kw):
    err = i32([0])
    got = decode(pool, q, table, ctx, layer=layer, err=err, **kw)
    want, pv, size = reference(pool, q, table, ctx, layer)
    assert int(err) == flag
    assert_within(got, want, bound(dtype, want, pv, size, P_ROUND[dtype]), "decode")
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,H,KV", [(64, 12, 12), (128, 4, 4), (64, 8, 2), (128, 32, 4), (64, 7, 1), (128, 9, 3),
                                     (64, 16, 1), (128, 24, 2), (64, 1, 1)])
def test_decode(dtype, hd, H, KV):
    """Lengths of zero and one, page borders and long ones; a middle layer; table entries behind a
    context hold ids outside the pool; NaN codes and NaN scales behind the last token and in pages not used."""
    rng = np.random.default_rng(hd + H)
    ctx = [1, 0, 15, 16, 17, 128, 129, 300, 1030, 0, 64]
    counts = [(n + PAGE - 1) // PAGE for n in ctx]
    P = sum(counts) + 5
    pool = Pool(P, 3, KV, hd, seed=H)
    table = tables(rng, counts, P)
    used = torch.zeros(P, dtype=torch.bool, device="cuda")
    for b, n in enumerate(ctx):
        for i in range(counts[b]):
            used[int(table[b, i])] = True
        if n % PAGE:
            page = int(table[b, counts[b] - 1])
            for t in (pool.k, pool.v):
                t[page, :, :, n % PAGE:] = 0x7f  # NaN
    for t in (pool.k, pool.v):
        t[~used] = 0x7f
    pool.k_scale[~used] = float("nan")
    q = torch.randn((len(ctx), H, hd), device="cuda", generator=torch.Generator(device="cuda").manual_seed(H)).to(DTYPES[dtype][1])
    got = check(pool, q, table, i32(ctx), 1, dtype)
    assert torch.equal(got[1], torch.zeros_like(got[1]))
    assert torch.equal(got, decode(pool, q, table, i32(ctx), layer=1))  # a fixed order of sums


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,H,KV,hd,n", [(1, 8, 8, 64, 5000), (2, 8, 1, 128, 20011), (1, 32, 8, 128, 40000), (70, 2, 2, 64, 333)])
def test_long_and_wide(dtype, B, H, KV, hd, n):
    rng = np.random.default_rng(n)
    ctx = [max(n - 7 * b, b) for b in range(B)]
    counts = [(c + PAGE - 1) // PAGE for c in ctx]
    pool = Pool(sum(counts), 1, KV, hd, seed=3)
    table = tables(rng, counts, sum(counts))
    q = torch.randn((B, H, hd), device="cuda").to(DTYPES[dtype][1])
    check(pool, q, table, i32(ctx), 0, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_peaked_and_shifted_scores(dtype):
    """Scores that rise along the context (the running maximum moves in every page), one token that takes
    all the weight, and blocks whose scales differ by many powers of two."""
    hd, H, KV = 64, 4, 2
    n = 400
    pool = Pool(25, 1, KV, hd, seed=1)
    table = i32([list(range(25))] * 3)
    order = torch.arange(25, device="cuda").float()
    pool.k_scale *= torch.exp2(order - 12)[:, None, None].clamp(2.0 ** -6, 2.0 ** 3)
    pool.v_scale *= torch.exp2(3 * (order % 7) - 9)[:, None, None]
    q = torch.randn((3, H, hd), device="cuda").to(DTYPES[dtype][1])
    q[1] *= 30
    q[2] *= 1e-3
    check(pool, q, table, i32([n, n - 3, n]), 0, dtype)


def test_small_values_keep_their_precision():
    """Values of 2^-40 and queries of 2^-30 and 2^40: nothing passes through a fixed-range 16-bit format."""
    hd, H, KV = 128, 2, 1
    for vs, qs, ks in ((2.0 ** -40, 1.0, 1.0), (2.0 ** 60, 2.0 ** -30, 2.0 ** 30), (1.0, 2.0 ** 40, 2.0 ** -40)):
        pool = Pool(8, 1, KV, hd, seed=2)
        pool.v_scale *= vs
        pool.k_scale *= ks
        table = i32([list(range(8))])
        q = torch.randn((1, H, hd), device="cuda") * qs
        check(pool, q, table, i32([121]), 0, "f32")


def test_nan_block_reaches_only_its_readers():
    hd, H, KV = 64, 2, 2
    pool = Pool(8, 1, KV, hd, seed=4)
    pool.k_scale[5, 0, 1] = float("nan")
    table = i32([[0, 1, 2, 3], [4, 5, 6, 7]])
    q = torch.randn((2, H, hd), device="cuda")
    got = decode(pool, q, table, i32([64, 60]))
    assert bool(got[1, 1].isnan().all()) and bool(got[0].isfinite().all()) and bool(got[1, 0].isfinite().all())


@pytest.mark.parametrize("B", [3, 64])
def test_bad_lengths_and_pages(B):
    """Too long, negative, and bad page ids: flagged, clamped or absent, the other rows unchanged."""
    hd, H, KV, width = 64, 4, 2, 8
    rng = np.random.default_rng(B)
    pool = Pool(B * width, 1, KV, hd, seed=6)
    table = tables(rng, [width] * B, B * width)
    ctx = rng.integers(1, width * PAGE + 1, B).tolist()
    q = torch.randn((B, H, hd), device="cuda")
    for b, n in ((0, width * PAGE + 1), (1, -5), (2, 2 ** 31 - 1)):
        c = list(ctx)
        c[b] = n
        check(pool, q, table, i32(c), 0, "f32", flag=2)
    for page in (-1, B * width, 2 ** 31 - 1):
        t, c = table.clone(), list(ctx)
        c[1] = width * PAGE - 3
        t[1, 2] = page
        check(pool, q, t, i32(c), 0, "f32", flag=2)
    t = table.clone()
    t[0] = -1
    c = list(ctx)
    c[0] = 100
    got = check(pool, q, t, i32(c), 0, "f32", flag=2)
    assert torch.equal(got[0], torch.zeros_like(got[0]))


def test_offsets_past_32_bits():
    """A pool of more than 2^32 codes: pages at its far end."""
    hd, H, KV, layers = 128, 8, 8, 4
    P = (1 << 32) // (layers * KV * PAGE * hd) + 20
    pool = Pool.__new__(Pool)
    pool.shape4 = (P, layers, KV, hd)
    for n in "kv":
        setattr(pool, n, torch.zeros((P, layers, KV, PAGE, hd), dtype=torch.uint8, device="cuda"))
        setattr(pool, n + "_scale", torch.ones((P, layers, KV), device="cuda"))
    small = Pool(16, layers, KV, hd, seed=8)
    for n in ("k", "v", "k_scale", "v_scale"):
        getattr(pool, n)[-16:] = getattr(small, n)
    q = torch.randn((1, H, hd), device="cuda")
    far = decode(pool, q, i32([list(range(P - 16, P))]), i32([250]), layer=3)
    assert torch.equal(far, decode(small, q, i32([list(range(16))]), i32([250]), layer=3))


def test_workspace_is_left_ready_and_can_be_shared_in_order():
    """Calls of different shapes one after another over one workspace; a captured graph replayed between them."""
    hd = 64
    size = max(lib().nr_paged_attention_kv8_workspace_size(b, h, kv, hd, w) for b, h, kv, w in ((1, 8, 8, 600), (40, 4, 1, 20)))
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    rng = np.random.default_rng(0)
    a = Pool(600, 1, 8, hd, seed=1), tables(rng, [600], 600), i32([9590]), torch.randn((1, 8, hd), device="cuda")
    b = Pool(800, 1, 1, hd, seed=2), tables(rng, [20] * 40, 800), i32(rng.integers(0, 321, 40).tolist()), torch.randn((40, 4, hd), device="cuda")
    want = [decode(p, q, t, c) for p, t, c, q in (a, b)]
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(a[3])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        decode(a[0], a[3], a[1], a[2], out=out, ws=ws)
    for _ in range(3):
        assert torch.equal(decode(b[0], b[3], b[1], b[2], ws=ws), want[1])
        out.zero_()
        graph.replay()
        assert torch.equal(out, want[0])
        assert torch.equal(decode(a[0], a[3], a[1], a[2], ws=ws), want[0])


@pytest.mark.parametrize("H,KV,hd", [(2, 2, 64), (16, 1, 128), (14, 2, 64)])
def test_long_contexts_of_few_sequences(H, KV, hd):
    """Items of many parts, one of few and an empty one in a wide table: a page outside the pool, then a
    NaN block, which reach their own sequence and heads only."""
    rng = np.random.default_rng(H)
    ctx = [5003, 0, 37, 4096, 1]
    counts = [(n + PAGE - 1) // PAGE for n in ctx]
    pool = Pool(sum(counts), 1, KV, hd, seed=H)
    table = tables(rng, counts, sum(counts))
    q = torch.randn((5, H, hd), device="cuda")
    sound = check(pool, q, table, i32(ctx), 0, "f32")
    bad = table.clone()
    bad[3, 100] = -1
    got = check(pool, q, bad, i32(ctx), 0, "f32", flag=2)
    assert torch.equal(got[:3], sound[:3]) and torch.equal(got[4], sound[4])
    pool.v_scale[int(table[0, 200]), 0, KV - 1] = float("nan")
    got = decode(pool, q, table, i32(ctx))
    assert bool(got[0, -(H // KV):].isnan().all()) and torch.equal(got[1:], sound[1:])
    assert torch.equal(got[0, :-(H // KV)], sound[0, :-(H // KV)])


def few_pages(B, KV, hd, ctx, width, seed, P=200):
    """A pool that many short contexts share, and tables into it of any pages."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = Pool(P, 1, KV, hd, seed=seed)
    return pool, torch.randint(0, P, (B, width), generator=g, device="cuda", dtype=torch.int32), i32(ctx)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,H,KV,hd,most", [(19, 16, 8, 128, 2100), (75, 4, 2, 64, 1500), (300, 3, 3, 64, 700)])
def test_many_items(dtype, B, H, KV, hd, most):
    """Over 148 (sequence, kv head) items, where a unit has 64 pages at least: contexts of several units,
    of one and of none side by side; those that pass a narrow table are clamped and flagged."""
    rng = np.random.default_rng(B)
    ctx = [most - 3, 0, 1, 1024, 1025] + rng.integers(0, most, B - 5).tolist()
    pool, table, lens = few_pages(B, KV, hd, ctx, (most + PAGE - 1) // PAGE, seed=B)
    q = torch.randn((B, H, hd), device="cuda").to(DTYPES[dtype][1])
    check(pool, q, table, lens, 0, dtype, flag=2 if max(ctx) > table.shape[1] * PAGE else 0)


def test_one_workspace_of_the_largest_batch():
    """A workspace sized for 1024 sequences of 17 kv heads, whose items are past the counters and stay
    uncut, serves smaller batches that are cut; what lies behind it is not touched."""
    H, KV, hd, width = 17, 17, 64, 130
    size = lib().nr_paged_attention_kv8_workspace_size(1024, H, KV, hd, width)
    ws = torch.zeros(size + 4096, dtype=torch.uint8, device="cuda")
    ws[size:] = 0xa5
    rng = np.random.default_rng(4)
    for B in (1024, 960, 30, 1):
        ctx = rng.integers(0, 60, B)
        ctx[0] = width * PAGE - 5
        pool, table, lens = few_pages(B, KV, hd, ctx.tolist(), width, seed=B, P=400)
        q = torch.randn((B, H, hd), device="cuda")
        got = decode(pool, q, table, lens, ws=ws)
        some = list(range(min(B, 40)))
        want, pv, size_ = reference(pool, q[some], table[some], lens[some], 0)
        assert_within(got[some], want, bound("f32", want, pv, size_, P_ROUND["f32"]), "decode")
        assert bool((ws[size:] == 0xa5).all())


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("B", [1, 5])  # parts joined by the second kernel, by an item's last CTA
@pytest.mark.parametrize("what", ["k_scale", "v_scale"])
def test_nan_block_of_no_weight(dtype, B, what):
    """A block with a NaN scale among tokens whose weights are 0 in fp32: its sequence and head are NaN
    however the context is cut, the others as without it."""
    hd, H, KV = 64, 16, 8
    ctx = [2000, 5, 1, 0, 33][:B]
    counts = [(n + PAGE - 1) // PAGE for n in ctx]
    pool = Pool(sum(counts), 1, KV, hd, seed=B)
    table = tables(np.random.default_rng(B), counts, sum(counts))
    q = torch.randn((B, H, hd), device="cuda", generator=torch.Generator(device="cuda").manual_seed(B))
    q[:, :, 0] = 8.0
    first = table[0, :8].long()  # scores of -112: weights of e^-112 and less
    pool.k[first] = 0
    pool.k[first, :, :, :, 0] = 0xfe  # -448
    pool.k_scale[first] = 0.25
    q = q.to(DTYPES[dtype][1])
    sound = check(pool, q, table, i32(ctx), 0, dtype)
    getattr(pool, what)[first[2], 0, 3] = float("nan")
    got = decode(pool, q, table, i32(ctx))
    assert bool(got[0, 6:8].isnan().all())
    got[0, 6:8] = sound[0, 6:8]
    assert torch.equal(got, sound)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,H,KV", [(64, 4, 2), (128, 12, 1)])
@pytest.mark.parametrize("large", [16.0, 2.0 ** 60])
def test_values_of_nothing_before_large_ones(dtype, hd, H, KV, large):
    """Blocks of zero values (scale 2^-126) with all the weight, then large values whose weights are 0 in
    fp32: no product of the two scales leaves the range."""
    pool = Pool(12, 1, KV, hd, seed=hd)
    table = i32([list(range(12))])
    q = torch.randn((1, H, hd), device="cuda", generator=torch.Generator(device="cuda").manual_seed(hd))
    q[:, :, 0] = 8.0
    q = q.to(DTYPES[dtype][1])
    pool.v[:8] = 0
    pool.v_scale[:8] = 2.0 ** -126
    pool.k[8:] = 0
    pool.k[8:, :, :, :, 0] = 0xfe  # -448: scores of -112 or -79, where the others are near 0
    pool.k_scale[8:] = 0.25
    pool.v_scale[8:] = large
    for first in (pool.v[:8], Pool(8, 1, KV, hd, seed=1).v):  # none, then values of 2^-117 and less
        pool.v[:8] = first
        got, (want, pv, size) = decode(pool, q, table, i32([12 * PAGE - 3])), reference(pool, q, table, [12 * PAGE - 3], 0)
        # weights are fp32 without its subnormals: what e^(s - m) < 2^-126 multiplies is lost, at most
        # 2^-126 sum |v|
        lost = 2.0 ** -126 * pool.values("v").abs().sum((0, 1, 3)).repeat_interleave(H // KV, 0)[None]
        assert_within(got, want, bound(dtype, want, pv, size, P_ROUND[dtype]) + lost, "decode")


def lost_weights(pool, q, table, ctx, layer):
    """What the weights' 16-bit form may lose: they enter the product in units in which the largest of
    p v_scale so far is at least 2^7, and an fp16 number is off by 2^-25 at most below its normal
    range: 2^-32 of the largest, of each |code|.  The second half of an fp32 weight is no finer there."""
    B, H, hd = q.shape
    KV = pool.shape4[2]
    out = torch.zeros((B, H, hd), dtype=torch.float64, device="cuda")
    for b in range(B):
        n = int(ctx[b])
        ids = table[b, :(n + PAGE - 1) // PAGE].long()
        for j in range(KV):
            kk = pool.values("k")[ids, layer, j].reshape(-1, hd)[:n]
            codes = pool.v[ids, layer, j].view(torch.float8_e4m3fn).double().reshape(-1, hd)[:n].abs().sum(0)
            vs = pool.v_scale[ids, layer, j].double().repeat_interleave(PAGE)[:n]
            g = H // KV
            p = torch.softmax(q[b, j * g:(j + 1) * g].double() @ kk.T / hd ** 0.5, -1)
            if n:
                out[b, j * g:(j + 1) * g] = 2.0 ** -32 * (p * vs).amax(-1, keepdim=True) * codes
    return out


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,H,KV", [(64, 4, 2), (128, 9, 1)])
def test_weights_far_below_the_largest(dtype, hd, H, KV):
    """Few tokens have nearly all the weight, and no values in half of the dims, where only tokens of
    weights down to 2^-60 of theirs count."""
    ctx = [7, 100, 333]
    pool = Pool(63, 1, KV, hd, seed=hd)
    g = torch.Generator(device="cuda").manual_seed(H)
    table = torch.arange(63, device="cuda", dtype=torch.int32).reshape(3, 21)
    q = torch.randn((3, H, hd), device="cuda", generator=g)
    q[:, :, 0] = 8.0
    q = q.to(DTYPES[dtype][1])
    pool.k[:, :, :, :, 0] = torch.randint(0x10, 0x7e, (63, 1, KV, PAGE), device="cuda", generator=g).to(torch.uint8) + 128
    pool.k[:, :, :, 3, 0] = 0
    pool.v[:, :, :, 3, :hd // 2] = 0
    got, (want, pv, size) = decode(pool, q, table, i32(ctx)), reference(pool, q, table, ctx, 0)
    assert_within(got, want, bound(dtype, want, pv, size, P_ROUND[dtype]) + lost_weights(pool, q, table, ctx, 0), "decode")


@pytest.mark.parametrize("B,H,KV,width", [(2, 16, 2, 200), (6, 8, 8, 200), (40, 8, 8, 80)])
def test_graph_replay_with_other_lengths(B, H, KV, width):
    """A captured call replayed with contexts and tables that were not there at the capture, on the
    paths of both joins and of whole items; two such graphs share a workspace, one after the other."""
    hd = 64
    rng = np.random.default_rng(B)
    pool, table, lens = few_pages(B, KV, hd, [1] * B, width, seed=B)
    q = torch.randn((B, H, hd), device="cuda")
    size = lib().nr_paged_attention_kv8_workspace_size(B, H, KV, hd, width)
    ws, outs = torch.zeros(size, dtype=torch.uint8, device="cuda"), [torch.zeros_like(q) for _ in range(2)]
    decode(pool, q, table, lens, out=outs[0], ws=ws)
    torch.cuda.synchronize()
    graphs = []
    for out in outs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            decode(pool, q, table, lens, out=out, ws=ws)
    for longest in (width * PAGE, 5, 0, width * PAGE - 7):
        lens.copy_(i32(rng.integers(0, longest + 1, B).tolist()))
        lens[-1] = longest
        table.copy_(table.flip(0).clone())
        for graph in graphs:
            graph.replay()
        want, pv, size_ = reference(pool, q, table, lens, 0)
        assert_within(outs[0], want, bound("f32", want, pv, size_, P_ROUND["f32"]), "replayed")
        assert torch.equal(outs[0], outs[1])
