"""nr_kv8_append against the formulas: rotation, scales, codes, what is left untouched."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from kv8_util import (DTYPES, E4M3, HALF, PAGE, Pool, append, assert_within, block_scale, e4m3, i32, rope, rotate,  # noqa: E402
                      tables)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for gpu tests")


def reference(pool, k32, v32, lens, start, table, layer):
    """The pool after the append, from rotated fp32 rows: one block at a time."""
    want = pool.clone()
    table = table.tolist()
    at = 0
    for b, n in enumerate(lens):
        p0 = start[b]
        for pg in range(p0 // PAGE, (p0 + n - 1) // PAGE + 1 if n else 0):
            lo, hi = max(p0, pg * PAGE), min(p0 + n, (pg + 1) * PAGE)
            page, had, slot = table[b][pg], (lo % PAGE if lo == p0 else 0), lo % PAGE
            for name, x in (("k", k32), ("v", v32)):
                blk = x[at + lo - p0:at + hi - p0].transpose(0, 1)  # [head, token, hd]
                codes, scales = getattr(want, name), getattr(want, name + "_scale")
                s = block_scale(blk.abs().amax((1, 2)))
                if had:
                    old = scales[page, layer]
                    new = torch.maximum(s, old)
                    moved = e4m3(codes[page, layer, :, :had].view(E4M3).float() * (old / new)[:, None, None]).view(torch.uint8)
                    grew = (new > old)[:, None, None]
                    codes[page, layer, :, :had] = torch.where(grew, moved, codes[page, layer, :, :had])
                    s = new
                codes[page, layer, :, slot:slot + hi - lo] = e4m3(blk / s[:, None, None]).view(torch.uint8)
                scales[page, layer] = s
        at += n
    return want


def same_pool(got, want):
    for n in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(got, n), getattr(want, n)), n


def case(seed, dtype, lens, start, H, KV, hd, layers=1, pad=0, scale=1.0):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [(p + n + PAGE - 1) // PAGE for n, p in zip(lens, start)]
    pool = Pool(sum(counts) + 3, layers, KV, hd, seed)
    table = tables(rng, counts, sum(counts) + 3)
    T = max(1, sum(lens) + pad)
    rows = (scale * torch.randn((T, (H + 2 * KV) * hd), generator=g, device="cuda")).to(DTYPES[dtype][1])
    cu = i32([0] + np.cumsum(lens).tolist())
    return pool, table, rows, cu, i32(start)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,H,KV,rot", [(64, 12, 12, 64), (128, 8, 2, 128), (128, 5, 5, 48), (64, 3, 1, 0), (64, 7, 7, 16)])
def test_append(dtype, layout, hd, H, KV, rot):
    """Ragged lengths from every kind of start, padding rows, a middle layer; q, k, v are
    column slices of one wider row."""
    lens = [1, 0, 17, 5, 16, 33, 1, 2, 40, 15]
    start = [0, 3, 15, 9, 16, 1, 31, 15, 30, 1]
    pool, table, rows, cu, st = case(hd + H + rot, dtype, lens, start, H, KV, hd, layers=3, pad=4)
    q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:]
    n = sum(lens)
    pos = torch.cat([torch.arange(p, p + m) for m, p in zip(lens, start)]).cuda()
    cos, sin = rope(80, rot)
    c, s = (cos[pos], sin[pos]) if rot else (None, None)
    split = lambda x, h: x[:n].reshape(n, h, hd)  # noqa: E731
    q32, k32 = (rotate(split(x, h).float(), c, s, rot, layout) for x, h in ((q, H), (k, KV)))
    want = reference(pool, k32, split(v, KV).float(), lens, start, table, 1)
    q_out = torch.full((len(rows), H * hd + 16), 7.0, dtype=rows.dtype, device="cuda")
    k_out = torch.full((len(rows), KV * hd), 7.0, dtype=rows.dtype, device="cuda")
    err = i32([0])
    for _ in range(2):  # appending the same tokens again changes nothing
        append(pool, q, k, v, cu, st, table, rot=rot, layout=layout, cos=cos, sin=sin, layer=1, n_heads=H,
               q_out=q_out[:, :H * hd], k_out=k_out, err=err)
        same_pool(pool, want)
    assert int(err) == 0
    assert torch.equal(q_out[:n, :H * hd], q32.to(rows.dtype).reshape(n, -1))
    assert torch.equal(k_out[:n], k32.to(rows.dtype).reshape(n, -1))
    assert bool((q_out[n:] == 7).all()) and bool((q_out[:, H * hd:] == 7).all()) and bool((k_out[n:] == 7).all())
    # and against 64 bits: the rotation to three fp32 roundings of terms up to |x1| + |x2|, then one of the type
    k64 = rotate(split(k, KV).double(), c, s, rot, layout)
    room = 2 * k64.abs().amax(-1, keepdim=True).expand_as(k64)
    tol = 3 * 2.0 ** -24 * room + HALF[dtype] * k64.abs()
    assert_within(k_out[:n].reshape(n, KV, hd), k64, tol, "rotated k")
    # a code is off by half a step of 3 bits, or of the subnormal spacing 2^-9
    got, at = pool.values("k"), 0
    for b, m in enumerate(lens):
        for i in range(m):
            p = start[b] + i
            page = int(table[b, p // PAGE])
            val, sc = got[page, 1, :, p % PAGE], pool.k_scale[page, 1].double()[:, None]
            x = k64[at + i]
            assert_within(val, x, torch.maximum(2.0 ** -4 * x.abs(), 2.0 ** -10 * sc) + 2.0 ** -4 * 3 * 2.0 ** -24 * room[at + i]
                          + 3 * 2.0 ** -24 * room[at + i], "k values")
        at += m


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_token_by_token_is_the_same_as_at_once(dtype):
    """Growing blocks: values get larger along the sequence, so scales grow several times within a
    page.  Values of full relative precision in every scale met keep their codes."""
    H, KV, hd, n = 2, 2, 64, 45
    pool, table, rows, cu, st = case(5, dtype, [n], [0], H, KV, hd)
    # magnitudes in [2^-2, 2^1.2]: no value falls below the normal range of the largest scale
    rows = (torch.sign(rows.float()) * (0.25 + rows.float().abs().clamp(max=1.0))
            * torch.linspace(1, 1.8, n, device="cuda")[:, None]).to(rows.dtype)
    q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:]
    one = pool.clone()
    append(pool, None, k, v, cu, st, table)
    for t in range(n):
        append(one, None, k[t:], v[t:], i32([0, 1]), i32([t]), table, T=1)
    same_pool(one, pool)


def test_in_place_and_without_outputs():
    H, KV, hd, rot = 4, 2, 128, 128
    lens, start = [20, 3], [4, 0]
    pool, table, rows, cu, st = case(9, "bf16", lens, start, H, KV, hd)
    cos, sin = rope(40, rot)
    other, plain = pool.clone(), rows.clone()
    parts = lambda r: (r[:, :H * hd], r[:, H * hd:(H + KV) * hd], r[:, (H + KV) * hd:])  # noqa: E731
    q, k, v = parts(rows)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    append(pool, q, k, v, cu, st, table, rot=rot, layout=1, cos=cos, sin=sin, n_heads=H, q_out=q_out, k_out=k_out)
    assert torch.equal(rows, plain)
    append(other, None, k, v, cu, st, table, rot=rot, layout=1, cos=cos, sin=sin)
    same_pool(other, pool)
    append(other, q, k, v, cu, st, table, rot=rot, layout=1, cos=cos, sin=sin, n_heads=H, q_out=q, k_out=k)
    same_pool(other, pool)
    assert torch.equal(q, q_out) and torch.equal(k, k_out) and torch.equal(v, parts(plain)[2])


@pytest.mark.parametrize("value", [0.0, 1e-42, 3e38, float("inf"), float("nan"), 448.0, 449.0, 2.0 ** -130])
def test_extreme_values(value):
    """All-zero, denormal and huge blocks, exact borders of a scale, and non-finite values: the block of
    a non-finite value gets a NaN scale, its neighbours do not."""
    KV, hd = 2, 64
    pool, table, rows, cu, st = case(3, "f32", [16, 16], [0, 0], 1, KV, hd, scale=0.0)
    k, v = rows[:, hd:hd + KV * hd], rows[:, hd + KV * hd:]
    k[3, 5] = value
    k[16:] = 1.0
    append(pool, None, k, v, cu, st, table)
    a, b = int(table[0, 0]), int(table[1, 0])
    got = pool.k_scale[a, 0, 0]
    want = block_scale(torch.tensor(abs(value), device="cuda"))
    assert torch.equal(got.isnan(), want.isnan()) and (bool(want.isnan()) or float(got) == float(want))
    assert float(pool.k_scale[a, 0, 1]) == 2.0 ** -126 and bool((pool.values("k")[a, 0, 1] == 0).all())
    assert bool((pool.values("k")[b] == 1.0).all())
    if np.isfinite(value):
        x = pool.values("k")[a, 0, 0, 3, 5].item()
        assert abs(x - k[3, 5].item()) <= max(2.0 ** -4 * abs(value), 2.0 ** -10 * float(want))


def test_out_of_range_is_skipped_and_flagged():
    """A sequence past its block table, past the rotation tables, with rows outside [0, T], at a negative
    position, and one with a bad page id: flagged, nothing of theirs written, the others as usual."""
    H = KV = 2
    hd, rot = 64, 64
    lens, start = [3, 20, 5, 2, 18], [2, 0, 30, 0, 8]
    pool, table, rows, cu, st = case(11, "bf16", lens, start, H, KV, hd)
    cos, sin = rope(60, rot)
    q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:]
    kw = dict(rot=rot, layout=0, cos=cos, sin=sin, n_heads=H)

    def go(cu, st, table, **more):
        p, e = pool.clone(), i32([0])
        qo, ko = torch.full_like(q, 9.0), torch.full_like(k, 9.0)
        append(p, q, k, v, cu, st, table, err=e, q_out=qo, k_out=ko, **{**kw, **more})
        return p, int(e), qo, ko

    good, e, qg, kg = go(cu, st, table)
    assert e == 0

    def without(b, p, qo, ko):
        lo, hi = int(cu[b]), int(cu[b + 1])
        assert bool((qo[lo:hi] == 9).all()) and bool((ko[lo:hi] == 9).all())
        keep = torch.ones(len(rows), dtype=torch.bool, device="cuda")
        keep[lo:hi] = False
        assert torch.equal(qo[keep], qg[keep]) and torch.equal(ko[keep], kg[keep])
        own = table[b, :(start[b] + lens[b] + 15) // 16].long()
        want = good.clone()
        for n in ("k", "v", "k_scale", "v_scale"):
            getattr(want, n)[own] = getattr(pool, n)[own]
        same_pool(p, want)

    for b, at in ((1, table.shape[1] * 16 - 19), (3, -1), (2, 2 ** 31 - 3)):
        bad = st.clone()
        bad[b] = at
        p, e, qo, ko = go(cu, bad, table)
        assert e == 2
        without(b, p, qo, ko)
    p, e, qo, ko = go(cu, st, table, rope_len=34)  # sequence 2 ends at 35
    assert e == 2
    without(2, p, qo, ko)
    p, e, qo, ko = go(cu, st, table, T=int(cu[-1]) - 1)  # the last sequence ends behind T
    assert e == 2
    without(4, p, qo, ko)
    for page in (-1, pool.shape4[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[4, 1] = page
        p, e, qo, ko = go(cu, st, t)
        assert e == 2 and torch.equal(qo, qg) and torch.equal(ko, kg)
        own = table[4, 1].long()
        want = good.clone()
        for n in ("k", "v", "k_scale", "v_scale"):
            getattr(want, n)[own] = getattr(pool, n)[own]
        same_pool(p, want)


def test_many_sequences_and_long_ones():
    """More sequences than one probe of the search covers, and sequences of many pages among empty ones."""
    rng = np.random.default_rng(2)
    KV, hd = 1, 64
    for lens in (rng.integers(0, 3, 1024).tolist(), [0] * 40 + [700] + [0] * 50 + [1, 333] + [0] * 3, [0, 0, 0]):
        start = rng.integers(0, 20, len(lens)).tolist()
        pool, table, rows, cu, st = case(7, "f16", lens, start, 1, KV, hd, pad=1)
        k, v = rows[:, hd:2 * hd], rows[:, 2 * hd:]
        n = sum(lens)
        want = reference(pool, k[:n].float().reshape(n, 1, hd), v[:n].float().reshape(n, 1, hd), lens, start, table, 0)
        append(pool, None, k, v, cu, st, table)
        same_pool(pool, want)


def test_graph_replay_and_other_stream():
    H, KV, hd, rot = 4, 4, 64, 64
    pool, table, rows, cu, st = case(21, "bf16", [1, 1, 1], [5, 16, 30], H, KV, hd)
    cos, sin = rope(64, rot)
    q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:]
    q_out, k_out = torch.zeros_like(q), torch.zeros_like(k)
    kw = dict(rot=rot, layout=1, cos=cos, sin=sin, n_heads=H, q_out=q_out, k_out=k_out)
    want = pool.clone()
    append(want, q, k, v, cu, st, table, **kw)
    first = q_out.clone()
    q_out.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        append(pool, q, k, v, cu, st, table, **kw)
    graph.replay()
    torch.cuda.synchronize()
    same_pool(pool, want)
    assert torch.equal(q_out, first)
    rows.mul_(2.0)  # replays read what is there now
    append(want, q, k, v, cu, st, table, **kw)
    second = q_out.clone()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        graph.replay()
    torch.cuda.synchronize()
    same_pool(pool, want)
    assert torch.equal(q_out, second)


def test_offsets_past_32_bits():
    """Pages at the far end of a pool of more than 2^32 codes, and rows past element 2^31 of their tensor."""
    H, KV, hd, layers, rot = 2, 8, 128, 4, 64
    P = (1 << 32) // (layers * KV * PAGE * hd) + 20
    pool = Pool.__new__(Pool)
    pool.shape4 = (P, layers, KV, hd)
    for n in "kv":
        setattr(pool, n, torch.zeros((P, layers, KV, PAGE, hd), dtype=torch.uint8, device="cuda"))
        setattr(pool, n + "_scale", torch.ones((P, layers, KV), device="cuda"))
    small = Pool(20, layers, KV, hd, zero=True)
    for n in "kv":
        getattr(small, n + "_scale").fill_(1.0)
    width = (H + 2 * KV) * hd
    rows = torch.zeros(((1 << 31) // width + 100, width), dtype=torch.bfloat16, device="cuda")
    lens, start = [37, 21], [5, 16]
    g = torch.Generator(device="cuda").manual_seed(1)
    rows[-sum(lens):] = torch.randn((sum(lens), width), generator=g, device="cuda").to(rows.dtype)
    cos, sin = rope(64, rot)
    cu = i32([0] + np.cumsum(lens).tolist())
    near = torch.arange(20, device="cuda", dtype=torch.int32).reshape(2, 10)
    kw = dict(rot=rot, layout=1, cos=cos, sin=sin, layer=3, n_heads=H)

    def go(p, rows, cu, table):
        q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + KV) * hd], rows[:, (H + KV) * hd:]
        err = i32([0])
        append(p, q, k, v, cu, i32(start), table, q_out=q, k_out=k, err=err, **kw)  # in place
        assert int(err) == 0

    last = rows[-sum(lens):].clone()
    go(small, last, cu, near)
    go(pool, rows, cu + (len(rows) - sum(lens)), near + (P - 20))
    assert torch.equal(rows[-sum(lens):], last)
    for n in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(pool, n)[-20:], getattr(small, n)), n
