"""The 8-bit page operators as a server uses them: prompts are turned and appended while prompt
attention answers them, then tokens follow one by one through append, decode attention and log
probabilities; every stage against 64 bits.  And the engine's own log probabilities."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from kv8_util import DTYPES, HALF, PAGE, Pool, append, assert_within, attend, bound, decode, i32, rope, rotate, stream, tables  # noqa: E402
from nitrorag_b200 import EngineConfig, NitroEngine, NrError  # noqa: E402
from nitrorag_b200._lib import lib  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def need_gpu():
    if not torch.cuda.is_available():
        pytest.fail("CUDA device required for gpu tests")


@pytest.mark.parametrize("dtype,hd,H,KV,layout", [("bf16", 128, 8, 2, 1), ("f16", 64, 3, 3, 0)])
def test_prompt_then_decode(dtype, hd, H, KV, layout):
    """Two layers share a pool; 3 prompts of different lengths, then 20 steps that cross page borders."""
    dt, layers, V, steps = DTYPES[dtype][1], 2, 1003, 20
    lens = [37, 128, 5]
    B, rot = len(lens), hd
    g = torch.Generator(device="cuda").manual_seed(hd)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    counts = [(n + steps + PAGE - 1) // PAGE for n in lens]
    pool = Pool(sum(counts) + 2, layers, KV, hd, zero=True)
    pool.k.fill_(0x7f)  # fresh pages hold anything
    pool.v.fill_(0x7f)
    table = tables(np.random.default_rng(1), counts, sum(counts) + 2)
    cos, sin = rope(max(lens) + steps, rot)
    head = rand(H * hd, V) / 8
    T = sum(lens)
    err = i32([0])
    keys = [[torch.zeros((0, KV, hd), dtype=torch.float64, device="cuda") for _ in range(B)] for _ in range(layers)]
    values = [[torch.zeros((0, KV, hd), dtype=torch.float64, device="cuda") for _ in range(B)] for _ in range(layers)]
    split = lambda x: (x[:, :H * hd], x[:, H * hd:(H + KV) * hd], x[:, (H + KV) * hd:])  # noqa: E731
    p_round = HALF[dtype] + 2.0 ** -13

    # prompts
    cu, start = i32([0] + np.cumsum(lens).tolist()), i32([0] * B)
    for layer in range(layers):
        rows = rand(T, (H + 2 * KV) * hd).to(dt)
        plain = rows.clone()
        q, k, v = split(rows)
        append(pool, q, k, v, cu, start, table, rot=rot, layout=layout, cos=cos, sin=sin, layer=layer, n_heads=H, q_out=q, k_out=k,
               err=err)  # in place
        out = torch.empty((T, H * hd), dtype=dt, device="cuda")
        rc = lib().nr_prompt_attention(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                       out.data_ptr(), out.stride(0), DTYPES[dtype][0], cu.data_ptr(), None, B, T, T, H, KV, hd,
                                       err.data_ptr(), stream())
        assert rc == 0
        for b, n in enumerate(lens):
            at = int(cu[b])
            k32 = rotate(split(plain)[1][at:at + n].reshape(n, KV, hd).float(), cos[:n], sin[:n], rot, layout)
            assert torch.equal(k[at:at + n], k32.to(dt).reshape(n, -1))
            keys[layer][b], values[layer][b] = k32.double(), v[at:at + n].reshape(n, KV, hd).double()
            seen = torch.ones((n, n), device="cuda").tril().bool()
            for h in range(H):
                j = h // (H // KV)
                cut = lambda x, i: x[at:at + n, i * hd:(i + 1) * hd].double()  # noqa: E731
                want, pv, size = attend(cut(q, h), cut(k, j), cut(v, j), seen)
                small = seen.double() @ cut(v, j).abs()
                assert_within(out[at:at + n, h * hd:(h + 1) * hd], want, bound(dtype, want, pv, size, p_round, small), "prompt")

    # tokens
    for step in range(steps):
        cu, start = i32(list(range(B + 1))), i32([n + step for n in lens])
        ctx = i32([n + step + 1 for n in lens])
        for layer in range(layers):
            rows = rand(B, (H + 2 * KV) * hd).to(dt)
            q, k, v = split(rows)
            pos = start.long()
            k32 = rotate(k.reshape(B, KV, hd).float(), cos[pos], sin[pos], rot, layout)
            append(pool, q, k, v, cu, start, table, rot=rot, layout=layout, cos=cos, sin=sin, layer=layer, n_heads=H, q_out=q, k_out=k,
                   err=err)
            qd = q.reshape(B, H, hd).contiguous()
            out = decode(pool, qd, table, ctx, layer=layer, err=err)
            for b in range(B):
                keys[layer][b] = torch.cat([keys[layer][b], k32[b:b + 1].double()])
                values[layer][b] = torch.cat([values[layer][b], v[b:b + 1].reshape(1, KV, hd).double()])
                n = int(ctx[b])
                ids = table[b, :(n + PAGE - 1) // PAGE].long()
                for j in range(KV):
                    kk, vv = (pool.values(x)[ids, layer, j].reshape(-1, hd)[:n] for x in "kv")
                    # what the pages hold: half a step of 3 bits, twice where a block's scale grew past a
                    # value's normal range (then at most the subnormal spacing of its block)
                    for got, exact, sc in ((kk, keys[layer][b][:, j], pool.k_scale), (vv, values[layer][b][:, j], pool.v_scale)):
                        s = sc[ids, layer, j].repeat_interleave(PAGE)[:n].double()[:, None]
                        assert_within(got, exact, torch.maximum(2.0 ** -4 * exact.abs(), 2.0 ** -10 * s) + 2.0 ** -10 * s, "pages")
                    gq = qd[b, j * (H // KV):(j + 1) * (H // KV)].double()
                    want, pv, size = attend(gq, kk, vv, torch.ones((len(gq), n), dtype=torch.bool, device="cuda"))
                    assert_within(out[b, j * (H // KV):(j + 1) * (H // KV)], want, bound(dtype, want, pv, size, 2.0 ** -11), "decode")
        logits = out.reshape(B, -1).float() @ head
        stats = [torch.zeros(s, dtype=d, device="cuda") for s, d in (((B,), torch.float32), ((B, 4), torch.float32), ((B, 4), torch.int32))]
        rc = lib().nr_token_logprobs(logits.data_ptr(), 0, V, B, V, None, 4, None, *(t.data_ptr() for t in stats), stream())
        assert rc == 0
        lp = torch.log_softmax(logits.double(), -1)
        assert torch.equal(stats[2], torch.topk(lp, 4, -1).indices.int())
        assert bool(((stats[1] - torch.topk(lp, 4, -1).values).abs() <= 2.0 ** -18 + 2.0 ** -23 * 20).all())
    assert int(err) == 0


def test_engine_last_decode_logprobs(tiny_model):
    """The engine's decode step, then its log probabilities from the logits it left on the GPU, against the
    logits it gave out; without logits, before a step and after a prefill they are refused."""
    eng = NitroEngine(tiny_model, EngineConfig(total_blocks=64, max_batch=8, max_prefill_tokens=64))
    rng = np.random.default_rng(3)
    with pytest.raises(NrError):
        eng.last_decode_logprobs(top_k=1)
    seqs, toks, pos = [], [], []
    for i in range(3):
        s = eng.seq_create(i)
        prompt = rng.integers(0, eng.vocab_size, 10 + 9 * i).astype(np.int32)
        _, t = eng.forward_prefill_chunk(s, prompt, 0)
        seqs.append(s), toks.append(t), pos.append(len(prompt))
    with pytest.raises(NrError):
        eng.last_decode_logprobs(top_k=1)
    eng.forward_decode_batch(toks, pos, seqs, want_logits=False)
    with pytest.raises(NrError):
        eng.last_decode_logprobs(top_k=1)
    for step in range(1, 3):
        lg, am = eng.forward_decode_batch(toks, [p + step for p in pos], seqs)
        targets = rng.integers(0, eng.vocab_size, 3)
        got = eng.last_decode_logprobs(targets, top_k=5)
        x = lg.astype(np.float64)
        lp = x - x.max(-1, keepdims=True)
        lp -= np.log(np.exp(lp).sum(-1, keepdims=True))
        order = np.argsort(-x, axis=-1, kind="stable")[:, :5]
        assert np.array_equal(got["top_ids"], order)
        tol = 2.0 ** -18 + 2.0 ** -23 * 40
        assert np.abs(got["top"] - np.take_along_axis(lp, order, 1)).max() <= tol
        assert np.abs(got["target"] - lp[np.arange(3), targets]).max() <= tol
        h = -(np.exp(lp) * lp).sum(-1)
        assert np.abs(got["entropy"] - h).max() <= 2.0 ** -18 * 12
        assert set(eng.last_decode_logprobs(top_k=0)) == {"entropy"}
        _, lg2 = eng.last_decode_outputs(want_logits=True)
        assert np.array_equal(lg, lg2)  # asking changed nothing
    with pytest.raises(NrError):
        eng.last_decode_logprobs(top_k=33)
    with pytest.raises(NrError):
        eng.last_decode_logprobs(targets=[0, 1])
    _, t = eng.forward_prefill_chunk(eng.seq_create(9), [1, 2, 3], 0)
    with pytest.raises(NrError):
        eng.last_decode_logprobs(top_k=1)
    eng.close()


def test_two_streams_at_once():
    """Prompts of both head sizes, decode and log probabilities on two streams side by side, each stream
    with its own workspace and outputs: what each gives alone."""
    g = torch.Generator(device="cuda").manual_seed(6)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    work = []
    for hd, H, KV, lens in ((64, 12, 12, [300, 41, 700]), (128, 8, 2, [513, 900])):
        B, T = len(lens), sum(lens)
        pool = Pool(40 * B, 1, KV, hd, seed=hd)
        work.append(dict(hd=hd, H=H, KV=KV, B=B, T=T, rows=rand(T, (H + 2 * KV) * hd).to(torch.bfloat16),
                         cu=i32([0] + np.cumsum(lens).tolist()), pool=pool, q=rand(B, H, hd).to(torch.bfloat16),
                         table=tables(np.random.default_rng(hd), [40] * B, 40 * B), ctx=i32([637 - 100 * b for b in range(B)]),
                         logits=rand(70, 32000), stream=torch.cuda.Stream()))

    def go(w):
        H, KV, hd = w["H"], w["KV"], w["hd"]
        q, k, v = w["rows"][:, :H * hd], w["rows"][:, H * hd:(H + KV) * hd], w["rows"][:, (H + KV) * hd:]
        out = torch.zeros((w["T"], H * hd), dtype=q.dtype, device="cuda")
        top, ids = torch.zeros((70, 4), device="cuda"), torch.zeros((70, 4), dtype=torch.int32, device="cuda")
        rc = lib().nr_prompt_attention(q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), out.data_ptr(),
                                       out.stride(0), 1, w["cu"].data_ptr(), None, w["B"], w["T"], w["T"], H, KV, hd, None, stream())
        rc |= lib().nr_token_logprobs(w["logits"].data_ptr(), 0, 32000, 70, 32000, None, 4, None, None, top.data_ptr(), ids.data_ptr(),
                                      stream())
        assert rc == 0
        return out, decode(w["pool"], w["q"], w["table"], w["ctx"]), top, ids

    want = [go(w) for w in work]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for i, w in enumerate(work):
            with torch.cuda.stream(w["stream"]):
                got.append((i, go(w)))
    torch.cuda.synchronize()
    for i, outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
