"""Plain 64-bit forms and helpers of the tests of the 8-bit page operators."""
import ctypes as C
import math

import torch

from nitrorag_b200._lib import NrKv8AppendArgs, NrKv8Pool, lib

DTYPES = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "f16": (2, torch.float16)}
E4M3 = torch.float8_e4m3fn
# half a step, relative to the value
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
PAGE = 16


def stream():
    return torch.cuda.current_stream().cuda_stream


def e4m3(x):
    return x.float().to(E4M3)


def block_scale(amax):
    """The smallest power of two >= 2^-126 with amax <= 448 * it (fp32 tensor in, fp32 out)."""
    f, e = torch.frexp(amax.float())
    s = torch.ldexp(torch.ones_like(f), e - 9 + (f > 0.875).int())
    s = torch.where(amax > 0, s, torch.zeros_like(s)).clamp(min=2.0 ** -126)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))


class Pool:
    """A device pool of random blocks (or zeros)."""

    def __init__(self, n_pages, n_layers, n_kv, hd, seed=0, zero=False):
        shape = (n_pages, n_layers, n_kv, PAGE, hd)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.shape4 = (n_pages, n_layers, n_kv, hd)
        for n in "kv":
            x = torch.zeros(shape, device="cuda") if zero else torch.randn(shape, generator=g, device="cuda")
            s = block_scale(x.abs().amax((-2, -1)))
            setattr(self, n, (x / s[..., None, None]).to(E4M3).view(torch.uint8))
            setattr(self, n + "_scale", s)

    def c(self):
        return NrKv8Pool(self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(), *self.shape4)

    def values(self, n):
        return getattr(self, n).view(E4M3).double() * getattr(self, n + "_scale").double()[..., None, None]

    def clone(self):
        p = Pool.__new__(Pool)
        p.shape4 = self.shape4
        for n in ("k", "v", "k_scale", "v_scale"):
            setattr(p, n, getattr(self, n).clone())
        return p


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tables(rng, counts, n_pages, width=None):
    """Disjoint pages from a shuffled pool; unused entries hold an id outside the pool."""
    perm = rng.permutation(n_pages).tolist()
    width = width or max(1, max(counts))
    t = [[n_pages + 7] * width for _ in counts]
    for b, n in enumerate(counts):
        for i in range(n):
            t[b][i] = perm.pop()
    return i32(t)


def rope(length, rot):
    if not rot:
        return None, None
    f = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") / (rot // 2))
    a = torch.arange(length, dtype=torch.float64, device="cuda")[:, None] * f
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def rotate(x, cos, sin, rot, layout):
    """x [n, heads, hd] in fp32 (the operator's arithmetic, each operation rounded) or 64 bits."""
    if not rot:
        return x.clone()
    y = x.clone()
    c, s = cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if layout == 0 else (i, i + rot // 2)
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def append(pool, q, k, v, cu, start, table, *, rot=0, layout=0, cos=None, sin=None, layer=0, n_heads=0, q_out=None,
           k_out=None, T=None, err=None, expect=0, rope_len=None):
    """nr_kv8_append over row tensors (possibly column slices of wider ones)."""
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[k.dtype]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    a = NrKv8AppendArgs(q=ptr(q), k=ptr(k), v=ptr(v), q_out=ptr(q_out), k_out=ptr(k_out), q_stride=ld(q), k_stride=ld(k),
                        v_stride=ld(v), q_out_stride=ld(q_out), k_out_stride=ld(k_out), cu_seqlens=cu.data_ptr(),
                        start_pos=start.data_ptr(), block_tables=table.data_ptr(), rope_cos=ptr(cos), rope_sin=ptr(sin),
                        dtype=code, B=len(start), T=len(k) if T is None else T, n_heads=n_heads,
                        max_pages=table.shape[1], layer=layer, rope_len=0 if cos is None else rope_len or len(cos),
                        rot_dim=rot, rope_layout=layout)
    p = pool.c()
    rc = lib().nr_kv8_append(C.byref(p), C.byref(a), ptr(err), stream())
    assert rc == expect
    return rc


def decode(pool, q, table, ctx, *, layer=0, out=None, ws=None, err=None, expect=0):
    """nr_paged_attention_decode_kv8; q [B, heads, hd]."""
    B, H, hd = q.shape
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[q.dtype]
    out = torch.full_like(q, float("nan")) if out is None else out
    if ws is None:
        size = lib().nr_paged_attention_kv8_workspace_size(B, H, pool.shape4[2], hd, table.shape[1])
        ws = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
    p = pool.c()
    rc = lib().nr_paged_attention_decode_kv8(q.data_ptr(), code, C.byref(p), layer, table.data_ptr(), table.shape[1],
                                             ctx.data_ptr(), B, H, out.data_ptr(), ws.data_ptr(),
                                             None if err is None else err.data_ptr(), stream())
    assert rc == expect
    return out


def attend(q, k, v, seen):
    """softmax(q k^T / sqrt(hd)) v in 64 bits, q [n, hd], k, v [m, hd], seen [n, m]; also sum p|v| and the
    largest |q|max * sum|k| / sqrt(hd), which the error bounds go by."""
    x = (q @ k.T / math.sqrt(q.shape[1])).masked_fill(~seen, -math.inf)
    p = torch.softmax(x, -1)
    p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
    size = q.abs().amax(-1) * k.abs().sum(-1).max() / math.sqrt(q.shape[1]) if len(k) else q.abs().amax(-1) * 0
    return p @ v, p @ v.abs(), size


def bound(dtype, out, pv, size, p_round, small=0.0):
    """|error| of an attention output: scores carry 2^-20 of |q|max sum|k| / sqrt(hd) (22-bit products of
    the split query, fp32 sums of up to 128 terms, the scale and log2 e factors), which moves a weight by
    that much relatively, twice with the normalisation; exp2 and sums 2^-17; weights rounded to the
    products' type (p_round); the output rounded once to its own.  fp16 values below 2^-14 are 2^-24
    apart, so there half a step is 2^-25 whatever the value: for the output, and for each weight
    (`small`: sum |v| over the keys seen, where weights enter a product as fp16 relative to a maximum near 1)."""
    rel = 2 * 2.0 ** -20 * size[..., None] + 2.0 ** -17 + p_round
    own = HALF[dtype] * out.abs()
    if dtype == "f16":
        own = own.clamp(min=2.0 ** -25) + 2.0 ** -25 * small
    return rel * pv + own + 1e-30


def assert_within(got, want, tol, what):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got[i].item()!r}, "
                             f"want {want[i].item()!r}, allowed {tol[i].item():.3e}")
