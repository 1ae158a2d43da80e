"""The serving operators over 8-bit K/V pages, as cases to measure: appending rotated keys
and values to the pages, decode attention that reads them, packed prompt attention and
token log probabilities.  ``run`` computes each either through the library's kernel-level
entry points (``own``) or in a plain form of elementary torch operations."""
import ctypes
import math
import random

import torch

own = False

PAGE = 16
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of one chat: the 110M model's heads, fp32 activations; pure latency
        dict(name="append_step_1", op="append", dtype="f32", heads=12, kv_heads=12, head_dim=64, rot=64, layout=0,
             seqs=1, lo=1, hi=1, past=700, pad=0, layers=1, mix=1),
        # one token for each of 64 running requests, grouped heads, a padded batch
        dict(name="append_step_64", op="append", dtype="bf16", heads=32, kv_heads=8, head_dim=128, rot=128, layout=1,
             seqs=61, lo=1, hi=1, past=2048, pad=3, layers=2, mix=2),
        # prompt chunks of several requests, packed, part of the head rotated
        dict(name="append_prompts", op="append", dtype="bf16", heads=32, kv_heads=8, head_dim=128, rot=64, layout=1,
             seqs=12, lo=33, hi=1300, past=600, pad=7, layers=1, mix=3),
        # one chat, 110M heads: latency
        dict(name="decode_1", op="decode", dtype="f32", heads=12, kv_heads=12, head_dim=64, seqs=1, lo=601, hi=601,
             layers=1, mix=4),
        # the paged attention microbenchmark's shape: 64 requests, contexts U[128, 1024]
        dict(name="decode_64", op="decode", dtype="f32", heads=12, kv_heads=12, head_dim=64, seqs=64, lo=128, hi=1024,
             layers=2, mix=5),
        # a busy server with grouped heads and contexts from empty to long
        dict(name="decode_grouped", op="decode", dtype="bf16", heads=32, kv_heads=8, head_dim=128, seqs=96, lo=0,
             hi=4096, layers=1, mix=6),
        # two very long contexts: few rows, a long axis
        dict(name="decode_long", op="decode", dtype="f16", heads=32, kv_heads=8, head_dim=128, seqs=2, lo=130000,
             hi=131072, layers=1, mix=7),
        # one short question
        dict(name="prompt_short", op="prompt", dtype="bf16", heads=12, kv_heads=12, head_dim=64, seqs=1, lo=37, hi=37,
             pad=0, mix=8),
        # ragged prompts of a batch, 110M heads
        dict(name="prompt_packed", op="prompt", dtype="f16", heads=12, kv_heads=12, head_dim=64, seqs=12, lo=17,
             hi=1000, pad=5, mix=9),
        # one long document, grouped heads
        dict(name="prompt_long", op="prompt", dtype="bf16", heads=32, kv_heads=8, head_dim=128, seqs=1, lo=8192,
             hi=8192, pad=0, mix=10),
        # the next token of 64 requests: log probabilities from the engine's fp32 logits, some words forbidden
        dict(name="score_step", op="score", dtype="f32", rows=64, vocab=32000, top=5, masked=True, mix=11),
        # scoring a prompt: every position's logits over a large vocabulary
        dict(name="score_prompt", op="score", dtype="bf16", rows=2048, vocab=128256, top=20, masked=False, mix=12),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt", "score"])
    mix = rng.randrange(1 << 30)
    head_dim = rng.choice([64, 128])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16])
    kv_heads = rng.randint(1, max(1, 32 // group))
    heads = group * kv_heads
    if op == "append":
        seqs = _between(rng, 1, 128)
        hi = 1 if rng.random() < 0.4 else _between(rng, 2, max(2, 8000 // seqs))
        return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rot=rng.choice([0, 16, 32, 48, 64, head_dim]), layout=rng.randint(0, 1), seqs=seqs,
                    lo=1 if hi == 1 else rng.choice([0, 1, hi // 2]), hi=hi, past=_between(rng, 1, 2000),
                    pad=rng.choice([0, 0, 1, 9]), layers=rng.randint(1, 3), mix=mix)
    if op == "decode":
        seqs = _between(rng, 1, 128)
        hi = _between(rng, 1, min(131072, (1 << 28) // (seqs * kv_heads * head_dim)))
        return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    seqs=seqs, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi,
                    layers=1 if seqs * hi > 20000 else rng.randint(1, 3), mix=mix)
    if op == "prompt":
        seqs = _between(rng, 1, 64)
        hi = _between(rng, 1, 8000 // seqs)
        return dict(op=op, dtype=rng.choice(["bf16", "f16"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    seqs=seqs, lo=rng.choice([0, 1, hi // 2, hi]), hi=hi, pad=rng.choice([0, 0, 3, 50]), mix=mix)
    rows = _between(rng, 1, 2048)
    vocab = _between(rng, 100, 128256)
    return dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]) if rows * vocab < 1 << 27 else "bf16", rows=rows,
                vocab=vocab, top=rng.choice([0, 1, 5, 8, 20]), masked=rng.random() < 0.3, mix=mix)


def _lengths(case):
    """Each sequence's new tokens (append, prompt) or context (decode), and its tokens before them."""
    rng = random.Random(case["mix"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    past = [rng.randint(0, case["past"]) for _ in lens] if "past" in case else [0] * len(lens)
    return lens, past


def work(case):
    if case["op"] == "score":
        m, v = case["rows"], case["vocab"]
        return {"bytes": m * v * BYTES[case["dtype"]] + m * (12 + 8 * case["top"]), "flops": 4.0 * m * v}
    lens, past = _lengths(case)
    h, g, d, e = case["heads"], case["kv_heads"], case["head_dim"], BYTES[case["dtype"]]
    t = sum(lens)
    if case["op"] == "append":
        # q, k, v in; q, k out; the codes of k and v and their blocks' scales
        blocks = sum((p + n + PAGE - 1) // PAGE - p // PAGE for n, p in zip(lens, past) if n)
        return {"bytes": t * d * e * (2 * h + 3 * g) + 2 * t * g * d + 8 * blocks * g, "flops": 3.0 * t * d * (h + 2 * g)}
    if case["op"] == "decode":
        blocks = sum((n + PAGE - 1) // PAGE for n in lens)
        return {"bytes": 2 * t * g * d + 8 * blocks * g + 2 * len(lens) * h * d * e, "flops": 4.0 * t * h * d}
    pairs = sum(n * (n + 1) // 2 for n in lens)
    return {"bytes": t * d * e * (2 * h + 2 * g), "flops": 4.0 * pairs * h * d}


# ------------------------------------------------------------------ inputs
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _quantize(x):
    """Blocks x [..., 16, d] of fp32 as e4m3 codes and one power-of-two scale for each block."""
    f, e = torch.frexp(x.abs().amax((-2, -1)))
    scale = torch.ldexp(torch.ones_like(f), e - 9 + (f > 0.875).int())
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def _pool(gen, n_pages, case):
    """Pages in use: codes and scales of normal values, some heads larger than others."""
    g, d, layers = case["kv_heads"], case["head_dim"], case["layers"]
    k_codes, k_scale, v_codes, v_scale = [], [], [], []
    step = max(1, (1 << 26) // (layers * g * PAGE * d))
    for at in range(0, n_pages, step):
        n = min(step, n_pages - at)
        for codes, scales in ((k_codes, k_scale), (v_codes, v_scale)):
            x = torch.randn((n, layers, g, PAGE, d), generator=gen, device="cuda")
            x *= torch.exp(0.5 * torch.randn((1, layers, g, 1, 1), generator=gen, device="cuda"))
            c, s = _quantize(x)
            codes.append(c)
            scales.append(s)
    return tuple(torch.cat([c.view(torch.uint8) if c.dtype == torch.float8_e4m3fn else c for c in p])
                 for p in (k_codes, k_scale, v_codes, v_scale))


def _tables(gen, pages_of, spare=3):
    """Block tables over a shuffled pool, and the pool's size."""
    most = max(1, max(pages_of))
    n_pages = sum(pages_of) + spare
    perm = torch.randperm(n_pages, generator=gen, device="cuda").int()
    table = torch.zeros((len(pages_of), most), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages_of):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, n_pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + case["mix"])
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "score":
        m, v = case["rows"], case["vocab"]
        s["logits"] = torch.empty((m, v), dtype=dt, device="cuda")
        step = max(1, (1 << 27) // v)
        for at in range(0, m, step):
            x = 2.5 * torch.randn((min(step, m - at), v), generator=gen, device="cuda")
            if case["masked"]:
                x[torch.rand(x.shape, generator=gen, device="cuda") < 0.3] = -math.inf
            s["logits"][at:at + step] = x.to(dt)
        s["targets"] = torch.randint(0, v, (m,), generator=gen, device="cuda", dtype=torch.int32)
        s["target_logprob"] = torch.zeros(m, device="cuda")
        s["entropy"] = torch.zeros(m, device="cuda")
        s["top_logprob"] = torch.zeros((m, case["top"]), device="cuda")
        s["top_ids"] = torch.zeros((m, case["top"]), dtype=torch.int32, device="cuda")
        return s
    lens, past = _lengths(case)
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    s["err"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    if case["op"] == "decode":
        s["q"] = torch.randn((len(lens), h, d), generator=gen, device="cuda").to(dt)
        s["out"] = torch.zeros_like(s["q"])
        s["table"], s["n_pages"] = _tables(gen, [(n + PAGE - 1) // PAGE for n in lens])
        s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"] = _pool(gen, s["n_pages"], case)
        s["ctx"] = _i32(lens)
        return s
    s["cu"] = _i32(cu)
    rows = max(1, cu[-1] + case["pad"])
    # one projection's output: q, k and v side by side in each row
    s["qkv"] = torch.randn((rows, (h + 2 * g) * d), generator=gen, device="cuda").to(dt)
    s["rows"] = rows
    if case["op"] == "prompt":
        s["out"] = torch.zeros((rows, h * d), dtype=dt, device="cuda")
        return s
    s["start"] = _i32(past)
    s["table"], s["n_pages"] = _tables(gen, [(p + n + PAGE - 1) // PAGE for n, p in zip(lens, past)])
    s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"] = _pool(gen, s["n_pages"], case)
    s["q_out"] = torch.zeros((rows, h * d), dtype=dt, device="cuda")
    s["k_out"] = torch.zeros((rows, g * d), dtype=dt, device="cuda")
    s["rope_len"] = max(p + n for n, p in zip(lens, past)) + 5
    if case["rot"]:
        half = case["rot"] // 2
        freq = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        angle = torch.arange(s["rope_len"], device="cuda", dtype=torch.float64)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ------------------------------------------------------------------ plain forms
def _split(s):
    c = s["case"]
    h, g, d = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"]
    return (x[:, :h * d].view(-1, h, d), x[:, h * d:(h + g) * d].view(-1, g, d), x[:, (h + g) * d:].view(-1, g, d))


def _rotate(x, cos, sin, rot, layout):
    """x [T, heads, d] fp32; cos, sin [T, rot/2]: two products and one sum for each element."""
    if not rot:
        return x
    y = x.clone()
    c, n = cos[:, None], sin[:, None]
    first = slice(0, rot, 2) if layout == 0 else slice(0, rot // 2)
    second = slice(1, rot, 2) if layout == 0 else slice(rot // 2, rot)
    a, b = x[..., first], x[..., second]
    y[..., first] = a * c - b * n
    y[..., second] = a * n + b * c
    return y


def _plain_append(s):
    c = s["case"]
    layer = c["layers"] - 1
    q, k, v = _split(s)
    rows = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    valid = rows < s["cu"][-1]
    seq = torch.searchsorted(s["cu"][1:], rows, right=True).clamp(max=c["seqs"] - 1)
    pos = torch.where(valid, s["start"][seq] + rows - s["cu"][seq], 0)
    cos = s["cos"][pos] if c["rot"] else None
    sin = s["sin"][pos] if c["rot"] else None
    q_rot = _rotate(q.float(), cos, sin, c["rot"], c["layout"])
    k_rot = _rotate(k.float(), cos, sin, c["rot"], c["layout"])
    # rows of the padding go to one page more than there are
    page = torch.where(valid, s["table"][seq, (pos // PAGE).clamp(max=s["table"].shape[1] - 1)], s["n_pages"]).long()
    slot = (pos % PAGE).long()
    first = s["start"][seq]
    goes_on = valid & (pos // PAGE == first // PAGE) & (first % PAGE > 0)
    out = []
    for x, codes, scales in ((k_rot, s["k_codes"], s["k_scale"]), (v.float(), s["v_codes"], s["v_scale"])):
        amax = torch.zeros((s["n_pages"] + 1, c["kv_heads"]), device="cuda")
        amax.scatter_reduce_(0, page[:, None].expand(-1, c["kv_heads"]), x.abs().amax(-1), "amax")
        f, e = torch.frexp(amax)
        fresh = torch.ldexp(torch.ones_like(f), e - 9 + (f > 0.875).int())
        fresh = torch.where(amax > 0, fresh, 0.0).clamp(min=2.0 ** -126)
        old_rows = torch.zeros(s["n_pages"] + 1, dtype=torch.int64, device="cuda")
        old_rows.scatter_reduce_(0, page, torch.where(goes_on, first % PAGE, 0).long(), "amax")
        started = old_rows > 0
        touched = torch.zeros(s["n_pages"] + 1, dtype=torch.bool, device="cuda")
        touched[page] = True
        before = scales[:, layer]
        after = torch.where(touched[:-1, None], torch.where(started[:-1, None], torch.maximum(before, fresh[:-1]), fresh[:-1]), before)
        # the rows that a block had before: coded anew where its scale grew
        grown = (started[:-1, None] & (after > before))[:, :, None, None]
        old = codes[:, layer].view(torch.float8_e4m3fn).float() * (before / after)[:, :, None, None]
        was = torch.arange(PAGE, device="cuda")[None] < old_rows[:-1, None]
        new = torch.where(grown & was[:, None, :, None], old.to(torch.float8_e4m3fn).view(torch.uint8), codes[:, layer])
        code = (x / torch.cat([after, after[:1]])[page][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        new = torch.cat([new, new[:1]])
        new[page, :, slot] = code
        codes = codes.clone()
        codes[:, layer] = new[:-1]
        scales = scales.clone()
        scales[:, layer] = after
        out += [codes.view(torch.float8_e4m3fn), scales]
    zero = torch.zeros((), device="cuda")
    q_rot = torch.where(valid[:, None, None], q_rot, zero).to(q.dtype).reshape(s["rows"], -1)
    k_rot = torch.where(valid[:, None, None], k_rot, zero).to(k.dtype).reshape(s["rows"], -1)
    return {"q": q_rot, "k": k_rot, "k_codes": out[0], "k_scale": out[1], "v_codes": out[2], "v_scale": out[3]}


def _softmax(x):
    """Over the last axis; rows that are -inf throughout give zeros."""
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    t = p.sum(-1, keepdim=True)
    return p / torch.where(t == 0, 1.0, t)


def _plain_decode(s):
    c = s["case"]
    layer, h, g, d = c["layers"] - 1, c["heads"], c["kv_heads"], c["head_dim"]
    table = s["table"].long()
    b, pages = table.shape
    seen = torch.arange(pages * PAGE, device="cuda")[None] < s["ctx"][:, None]
    kv = []
    for codes, scales in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])):
        x = codes[:, layer][table].view(torch.float8_e4m3fn).float() * scales[:, layer][table][..., None, None]
        kv.append(x.permute(0, 2, 1, 3, 4).reshape(b, g, pages * PAGE, d))
    q = s["q"].float().view(b, g, h // g, d)
    x = torch.matmul(q, kv[0].transpose(2, 3)) * (1.0 / math.sqrt(d))
    p = _softmax(torch.where(seen[:, None, None], x, -math.inf))
    out = torch.matmul(p, torch.where(seen[:, None, :, None], kv[1], 0.0))
    return out.reshape(b, h, d).to(s["q"].dtype)


def _plain_prompt(s):
    c = s["case"]
    h, g, d, t = c["heads"], c["kv_heads"], c["head_dim"], s["rows"]
    q, k, v = (x.float().transpose(0, 1) for x in _split(s))
    rows = torch.arange(t, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["cu"][1:], rows, right=True)
    valid = rows < s["cu"][-1]
    seen = (seq[:, None] == seq[None]) & (rows[None] <= rows[:, None]) & valid[:, None] & valid[None]
    x = torch.matmul(q.reshape(g, h // g * t, d), k.transpose(1, 2)).view(g, h // g, t, t)
    x.mul_(1.0 / math.sqrt(d)).masked_fill_(~seen, -math.inf)
    out = torch.matmul(_softmax(x).view(g, h // g * t, t), v).view(h, t, d)
    return out.transpose(0, 1).reshape(t, h * d).to(s["qkv"].dtype)


def _plain_score(s):
    c = s["case"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    t = e.sum(-1, keepdim=True)
    lp = y - torch.log(t)
    entropy = torch.log(t[:, 0]) - (e * torch.where(e > 0, y, 0.0)).sum(-1) / t[:, 0]
    out = {"target_logprob": lp.gather(1, s["targets"].long()[:, None])[:, 0], "entropy": entropy}
    if c["top"]:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        out |= {"top_logprob": lp.gather(1, ids), "top_ids": ids.int()}
    return out


# ------------------------------------------------------------------ the library's operators
def _bind(s):
    """The call a program makes each step, with the addresses that stay the same."""
    from nitrorag_b200 import _lib
    c, lib = s["case"], _lib.lib()
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["op"] == "score":
        top = c["top"]
        return lib.nr_token_logprobs, (p["logits"], CODES[c["dtype"]], c["vocab"], c["rows"], c["vocab"], p["targets"], top,
                                       p["target_logprob"], p["entropy"], p["top_logprob"] if top else None,
                                       p["top_ids"] if top else None)
    h, g, d = c["heads"], c["kv_heads"], c["head_dim"]
    e = BYTES[c["dtype"]]
    if c["op"] == "prompt":
        stride = (h + 2 * g) * d
        return lib.nr_prompt_attention, (p["qkv"], stride, p["qkv"] + h * d * e, stride, p["qkv"] + (h + g) * d * e, stride,
                                         p["out"], h * d, CODES[c["dtype"]], p["cu"], None, c["seqs"], s["rows"], s["rows"],
                                         h, g, d, p["err"])
    pool = _lib.NrKv8Pool(p["k_codes"], p["v_codes"], p["k_scale"], p["v_scale"], s["n_pages"], c["layers"], g, d)
    if c["op"] == "decode":
        size = lib.nr_paged_attention_kv8_workspace_size(c["seqs"], h, g, d, s["table"].shape[1])
        s["workspace"] = torch.zeros(size, dtype=torch.uint8, device="cuda")
        return lib.nr_paged_attention_decode_kv8, (p["q"], CODES[c["dtype"]], ctypes.byref(pool), c["layers"] - 1, p["table"],
                                                   s["table"].shape[1], p["ctx"], c["seqs"], h, p["out"],
                                                   s["workspace"].data_ptr(), p["err"])
    stride = (h + 2 * g) * d
    args = _lib.NrKv8AppendArgs(
        q=p["qkv"], k=p["qkv"] + h * d * e, v=p["qkv"] + (h + g) * d * e, q_out=p["q_out"], k_out=p["k_out"],
        q_stride=stride, k_stride=stride, v_stride=stride, q_out_stride=h * d, k_out_stride=g * d,
        cu_seqlens=p["cu"], start_pos=p["start"], block_tables=p["table"], rope_cos=p.get("cos"), rope_sin=p.get("sin"),
        dtype=CODES[c["dtype"]], B=c["seqs"], T=s["rows"], n_heads=h, max_pages=s["table"].shape[1], layer=c["layers"] - 1,
        rope_len=s["rope_len"], rot_dim=c["rot"], rope_layout=c["layout"])
    return lib.nr_kv8_append, (ctypes.byref(pool), ctypes.byref(args), p["err"])


def run(state):
    op = state["case"]["op"]
    if own:
        if "call" not in state:
            state["call"] = _bind(state)
        call, args = state["call"]
        status = call(*args, torch.cuda.current_stream().cuda_stream)
        if status < 0:
            raise RuntimeError("%s: status %d" % (op, status))
        if op == "append":
            return {"q": state["q_out"], "k": state["k_out"], "k_codes": state["k_codes"].view(torch.float8_e4m3fn),
                    "k_scale": state["k_scale"], "v_codes": state["v_codes"].view(torch.float8_e4m3fn), "v_scale": state["v_scale"]}
        if op == "score":
            names = ["target_logprob", "entropy"] + (["top_logprob", "top_ids"] if state["case"]["top"] else [])
            return {n: state[n] for n in names}
        return state["out"]
    if op == "append":
        return _plain_append(state)
    if op == "decode":
        return _plain_decode(state)
    if op == "prompt":
        return _plain_prompt(state)
    return _plain_score(state)


# ------------------------------------------------------------------ the definition, in 64 bits
def _exact_append(s):
    """Sequence by sequence and block by block."""
    c = s["case"]
    layer, rot = c["layers"] - 1, c["rot"]
    lens, past = _lengths(c)
    q, k, v = (x.double() for x in _split(s))
    table = s["table"].cpu()
    out = {"q": torch.zeros_like(q), "k": torch.zeros_like(k)}
    pools = {n: s[n + "_codes"].view(torch.float8_e4m3fn).double() for n in "kv"}
    scales = {n: s[n + "_scale"].double() for n in "kv"}
    at = 0
    for b, (n, p) in enumerate(zip(lens, past)):
        if not n:
            continue
        turned = {}
        for name, x in (("q", q), ("k", k)):
            x = x[at:at + n].clone()
            if rot:
                z = torch.complex(s["cos"][p:p + n].double(), s["sin"][p:p + n].double())[:, None]
                if c["layout"] == 0:
                    w = torch.view_as_complex(x[..., :rot].reshape(n, -1, rot // 2, 2).contiguous()) * z
                    x[..., :rot] = torch.view_as_real(w).reshape(n, -1, rot)
                else:
                    w = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * z
                    x[..., :rot] = torch.cat([w.real, w.imag], -1)
            out[name][at:at + n] = x
            turned[name] = x
        for name, x in (("k", turned["k"]), ("v", v[at:at + n])):
            for page in range(p // PAGE, (p + n - 1) // PAGE + 1):
                lo, hi = max(p, page * PAGE), min(p + n, (page + 1) * PAGE)
                have = lo % PAGE if lo == p else 0
                block = x[lo - p:hi - p].transpose(0, 1)  # [head, token, d]
                i = int(table[b, page])
                top = block.abs().amax((1, 2))
                scale = torch.exp2(torch.ceil(torch.log2((top / 448.0).clamp(min=2.0 ** -126))))
                if have:
                    scale = torch.maximum(scale, scales[name][i, layer])
                    pools[name][i, layer, :, :have] *= (scales[name][i, layer] / scale)[:, None, None]
                pools[name][i, layer, :, lo % PAGE:lo % PAGE + hi - lo] = block / scale[:, None, None]
                scales[name][i, layer] = scale
        at += n
    for name in "kv":
        out[name + "_codes"] = pools[name].float().to(torch.float8_e4m3fn).double()
        out[name + "_scale"] = scales[name]
    out["q"], out["k"] = out["q"].flatten(1), out["k"].flatten(1)
    return out


def _exact_decode(s):
    c = s["case"]
    layer, h, g, d = c["layers"] - 1, c["heads"], c["kv_heads"], c["head_dim"]
    lens, _ = _lengths(c)
    out = torch.zeros((len(lens), h, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        if not n:
            continue
        pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
        k, v = (s[x + "_codes"][pages, layer].view(torch.float8_e4m3fn).double() * s[x + "_scale"][pages, layer, :, None, None].double()
                for x in "kv")
        for j in range(h):
            kj, vj = k[:, j * g // h].reshape(-1, d)[:n], v[:, j * g // h].reshape(-1, d)[:n]
            out[b, j] = torch.softmax(kj @ s["q"][b, j].double() / math.sqrt(d), 0) @ vj
    return out


def _exact_prompt(s):
    c = s["case"]
    h, g, d = c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = (x.double() for x in _split(s))
    out = torch.zeros((s["rows"], h, d), dtype=torch.float64, device="cuda")
    at = 0
    for n in _lengths(c)[0]:
        future = torch.ones((n, n), dtype=torch.bool, device="cuda").triu(1)
        for j in range(h if n else 0):
            x = q[at:at + n, j] @ k[at:at + n, j * g // h].T / math.sqrt(d)
            out[at:at + n, j] = torch.softmax(x.masked_fill_(future, -math.inf), -1) @ v[at:at + n, j * g // h]
        at += n
    return out.flatten(1)


def _exact_score(s):
    c = s["case"]
    got = {"target_logprob": [], "entropy": [], "top_logprob": []}
    step = max(1, (1 << 26) // c["vocab"])
    for at in range(0, c["rows"], step):
        lp = torch.log_softmax(s["logits"][at:at + step].double(), -1)
        got["target_logprob"].append(lp[torch.arange(len(lp), device="cuda"), s["targets"][at:at + step].long()])
        got["entropy"].append(-torch.xlogy(lp.exp(), lp.exp()).sum(-1))
        got["top_logprob"].append(torch.topk(lp, c["top"], -1).values if c["top"] else lp[:, :0])
    got = {n: torch.cat(v) for n, v in got.items()}
    if c["top"]:
        return got | {"top_ids": None}
    del got["top_logprob"]
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "prompt": _exact_prompt, "score": _exact_score}[case["op"]](s)
