"""Norm of queries and keys with the rotation of their positions, and its gradient (GPU), against
the formulas in 64 bits.

Tolerances. u = half a step of the storage type (2^-8 bf16, 2^-11 fp16), f = 2^-24 that of fp32. The
kernels compute in fp32 and round once:
  y:  u |y| + 2^-18 m, m = the row's largest |x^ w| + |b|: 64 f for the sums over a row (at most 32
      additions in a lane and 10 across lanes, half of that after the square root), the mean's
      subtraction, the products and the turn; and 2^-25, half the step below fp16's normal range.
  dx: u |dx| + 2^-17 r (max|d| + max|x^| |mean(d x^)| + |mean(d)|), the same with one more sum.
  dw, db: fp32 sums of at most 64 rows in a lane and 16 joins, then 64 bits: 2^-17 of sum |g x^|.
"""
import pytest
import torch

import mod_dit_amd as md
from mod_dit_amd import ops

pytestmark = pytest.mark.gpu


def _tensor(B, H, S, D, dtype, nhd, g, scale=1.0):
    t = (torch.randn((B, S, H, D) if nhd else (B, H, S, D), generator=g) * scale).to(dtype).cuda()
    return t.transpose(1, 2) if nhd else t


def _tables(n, D, full, batch, g):
    a = torch.rand((batch, n, D // 2) if batch else (n, D // 2), generator=g, dtype=torch.float64) * 6.28
    c, s = a.cos().float(), a.sin().float()
    if full == "interleaved":
        c, s = c.repeat_interleave(2, -1), s.repeat_interleave(2, -1)
    elif full == "halves":
        c, s = torch.cat([c, c], -1), torch.cat([s, s], -1)
    return c.cuda(), s.cuda()


def _setup(B, H, Sq, Sk, D, dtype, nhd, norm, across, tables, offset, rotated, affine, w_dtype, batch_tables=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = _tensor(B, H, Sq, D, dtype, nhd, g, 3.0)
    k = _tensor(B, H, Sk, D, dtype, nhd, g, 0.3) + 0.5
    kw = dict(norm=norm, across_heads=across, eps=1e-5, rope_offset=offset, interleaved=tables != "halves")
    n = D * (H if across else 1)
    if norm != "none":
        for name, on in (("q_weight", "w" in affine), ("k_weight", "w" in affine),
                         ("q_bias", "b" in affine), ("k_bias", "b" in affine)):
            kw[name] = (torch.randn(n, generator=g) + ("weight" in name)).to(w_dtype).cuda() if on else None
    if rotated:
        half = tables.startswith("half_")
        kw["interleaved"] = tables in ("interleaved", "half_interleaved")
        kw["cos"], kw["sin"] = _tables(rotated, D, "" if half else tables, batch_tables and B, g)
    return q, k, kw


def _norm64(x, kw):
    """(x^, r, the dims normed over) of fp64 x."""
    if kw["norm"] == "none":
        return x, torch.ones_like(x[..., :1]), (3,)
    over = (1, 3) if kw["across_heads"] else (3,)
    if kw["norm"] == "layer":
        x = x - x.mean(over, keepdim=True)
    r = (x.square().mean(over, keepdim=True) + kw["eps"]).rsqrt()
    return x * r, r, over


def _shaped(t, x, kw, none):
    if t is None:
        return torch.full_like(x[:1, :, :1], none)
    t = t.double()
    return t.view(1, x.shape[1], 1, x.shape[3]) if kw["across_heads"] else t


def _turn64(x, kw, back=False):
    cos, sin = kw.get("cos"), kw.get("sin")
    if cos is None:
        return x
    D, n, off = x.shape[-1], cos.shape[-2], kw["rope_offset"]
    i = torch.arange(D // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if kw["interleaved"] else (i, i + D // 2)
    ci, si = (a, b) if cos.shape[-1] == D else (i, i)
    c, s = cos.double()[..., ci], sin.double()[..., si]
    if cos.ndim == 3:
        c, s = c[:, None], s[:, None]
    s = -s if back else s
    t = slice(off, off + n)
    y = x.clone()
    y[:, :, t, a] = x[:, :, t, a] * c - x[:, :, t, b] * s
    y[:, :, t, b] = x[:, :, t, b] * c + x[:, :, t, a] * s
    return y


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _check_forward(got, x, w, b, kw):
    n, _, over = _norm64(x.double(), kw)
    y = n * _shaped(w, n, kw, 1.0) + _shaped(b, n, kw, 0.0)
    m = (n * _shaped(w, n, kw, 1.0)).abs().amax(over, keepdim=True) + _shaped(b, n, kw, 0.0).abs()
    y = _turn64(y, kw)
    tol = _half(x.dtype) * y.abs() + 2.0 ** -18 * m.amax(-1, keepdim=True) + 2.0 ** -25
    assert got.dtype == x.dtype and got.shape == x.shape
    assert ((got.double() - y).abs() <= tol).all(), ((got.double() - y).abs() / tol).max()


def _grads64(x, dy, w, b, kw):
    """(dx, dw, db) and the tolerances of each."""
    x, dy = x.double(), dy.double()
    g = _turn64(dy, kw, back=True)
    if kw["norm"] == "none":
        return (g, None, None), (2.0 ** -22 * dy.abs().amax(-1, keepdim=True), None, None)
    n, r, over = _norm64(x, kw)
    d = g * _shaped(w, n, kw, 1.0)
    m2 = (d * n).mean(over, keepdim=True)
    m1 = d.mean(over, keepdim=True) if kw["norm"] == "layer" else torch.zeros_like(m2)
    rows = (0, 2) if kw["across_heads"] else (0, 1, 2)
    top = lambda t: t.abs().amax(over, keepdim=True)  # noqa: E731
    tol = 2.0 ** -17 * r * (top(d) + top(n) * m2.abs() + m1.abs())
    return (((d - n * m2 - m1) * r, (g * n).sum(rows).flatten(), g.sum(rows).flatten()),
            (tol, 2.0 ** -17 * (g * n).abs().sum(rows).flatten(), 2.0 ** -17 * g.abs().sum(rows).flatten()))


def _check_grads(got, x, dy, w, b, kw):
    want, tol = _grads64(x, dy, w, b, kw)
    lim = _half(x.dtype) * want[0].abs() + tol[0] + 2.0 ** -25
    assert got[0].dtype == x.dtype
    assert ((got[0].double() - want[0]).abs() <= lim).all(), ((got[0].double() - want[0]).abs() / lim).max()
    for t, at in ((w, 1), (b, 2)):
        if t is None:
            assert got[at] is None
            continue
        assert got[at].dtype == torch.float32 and got[at].shape == t.shape
        assert ((got[at].double() - want[at]).abs() <= tol[at]).all()


BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
# B, H, Sq, Sk, D, dtype, nhd, norm, across, tables, offset, rotated, affine, weights' dtype
CASES = [
    (1, 1, 1, 1, 64, BF, False, "rms", False, "interleaved", 0, 1, "w", F32),
    (1, 24, 1, 1, 128, BF, True, "rms", False, "interleaved", 0, 1, "w", BF),
    (2, 3, 77, 77, 128, BF, True, "rms", False, "halves", 0, 77, "w", BF),
    (2, 5, 130, 130, 64, FP, False, "layer", False, "interleaved", 31, 99, "wb", FP),
    (1, 2, 200, 9, 128, FP, False, "layer", False, "half_interleaved", 2, 5, "w", F32),   # q longer than k
    (1, 7, 33, 64, 64, BF, True, "rms", False, "half_halves", 33, 0, "", F32),            # nothing rotated
    (1, 3, 65, 65, 128, BF, False, "none", False, "half_halves", 10, 40, "", F32),
    (1, 4, 50, 50, 64, FP, True, "none", False, "interleaved", 0, 50, "", F32),
    (1, 5, 19, 19, 128, BF, True, "rms", True, "interleaved", 0, 19, "w", BF),
    (2, 40, 21, 20, 128, BF, True, "rms", True, "halves", 3, 17, "w", F32),
    (1, 64, 9, 9, 128, FP, False, "layer", True, "interleaved", 0, 9, "wb", FP),          # the widest row
    (1, 1, 70, 70, 64, BF, False, "layer", True, "half_interleaved", 69, 1, "wb", BF),
    (1, 20, 40, 40, 64, BF, True, "rms", True, "interleaved", 0, 40, "w", F32),
    (1, 48, 1100, 1100, 64, FP, False, "layer", False, "interleaved", 226, 874, "wb", FP),
    (1, 24, 1500, 1500, 128, BF, True, "rms", False, "interleaved", 0, 1500, "w", BF),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("batch_tables", [0, 1])
def test_values_and_gradients(case, batch_tables):
    q, k, kw = _setup(*case, batch_tables=batch_tables)
    w, b = [kw.get("q_weight"), kw.get("k_weight")], [kw.get("q_bias"), kw.get("k_bias")]
    got = ops.qk_norm_rope(q, k, **kw)
    for y, x, wi, bi in zip(got, (q, k), w, b):
        _check_forward(y, x, wi, bi, kw)
    g = torch.Generator().manual_seed(9)
    dq, dk = (torch.randn(t.shape, generator=g).to(t.dtype).cuda() for t in (q, k))
    res = ops.qk_norm_rope_bwd(q, k, dq, dk, **kw)
    again = ops.qk_norm_rope_bwd(q, k, dq, dk, **kw)
    for a, c in zip(res, again):
        assert (a is None and c is None) or torch.equal(a, c)
    _check_grads((res[0], res[2], res[4]), q, dq, w[0], b[0], kw)
    _check_grads((res[1], res[3], res[5]), k, dk, w[1], b[1], kw)


@pytest.mark.parametrize("norm,across", [("rms", False), ("layer", False), ("rms", True), ("layer", True)])
def test_gradients_against_differences(norm, across):
    """The kernel's gradient along random directions against central differences of the 64-bit
    formula; the tolerance adds the gradients' own."""
    q, k, kw = _setup(1, 3, 40, 40, 64, BF, True, norm, across, "interleaved", 5, 30, "wb", F32)
    w, b = kw["q_weight"], kw["q_bias"]
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(q.shape, generator=g).to(BF).cuda()
    got = ops.qk_norm_rope_bwd(q, k, dy, torch.zeros_like(k), **kw)
    got = (got[0], got[2], got[4])
    want, tol = _grads64(q, dy, w, b, kw)
    f = lambda x, w, b: (_turn64(_norm64(x, kw)[0] * _shaped(w, x, kw, 1.0)  # noqa: E731
                                 + _shaped(b, x, kw, 0.0), kw) * dy.double()).sum()
    at = [t.double() for t in (q, w, b)]
    for i in range(3):
        v = torch.randn(at[i].shape, generator=g, dtype=torch.float64).cuda()
        h = 1e-5
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + h * v, at[i] - h * v
        diff = ((f(*plus) - f(*minus)) / (2 * h)).item()
        lim = tol[i] + (_half(BF) * want[0].abs() if i == 0 else 0.0)
        # the difference itself: h^2 of third derivatives and 1e-16 / h of f
        assert abs((got[i].double() * v).sum().item() - diff) <= (v.abs() * lim).sum().item() + 1e-6 * abs(diff) + 1e-6


def test_in_place_and_into_slices():
    """out may be q and k themselves, or parts of a longer sequence whose other rows stay."""
    q, k, kw = _setup(1, 4, 100, 100, 128, BF, False, "rms", False, "interleaved", 0, 100, "w", BF)
    want = ops.qk_norm_rope(q, k, **kw)
    joint = torch.full((2, 1, 4, 130, 128), 7.0, dtype=BF, device="cuda")
    ops.qk_norm_rope(q, k, out=(joint[0, :, :, 17:117], joint[1, :, :, 17:117]), **kw)
    assert torch.equal(joint[0, :, :, 17:117], want[0]) and torch.equal(joint[1, :, :, 17:117], want[1])
    assert (joint[:, :, :, :17] == 7).all() and (joint[:, :, :, 117:] == 7).all()
    a, b = q.clone(), k.clone()
    got = ops.qk_norm_rope(a, b, out=(a, b), **kw)
    assert got[0] is a and torch.equal(a, want[0]) and torch.equal(b, want[1])
    q, k, kw = _setup(1, 4, 100, 100, 128, BF, True, "rms", True, "interleaved", 0, 100, "w", BF)
    want = ops.qk_norm_rope(q, k, **kw)
    ops.qk_norm_rope(q, k, out=(q, k), **kw)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_fused_projection_slices_and_broadcast_rows():
    """q and k as slices of one projection; a batch that is expanded, not stored."""
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn((2, 60, 3, 5, 64), generator=g).to(BF).cuda()
    q, k = (qkv[:, :, i].transpose(1, 2) for i in (0, 1))
    w = torch.randn(64, generator=g).cuda()
    want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), q_weight=w, k_weight=w)
    got = ops.qk_norm_rope(q, k, q_weight=w, k_weight=w)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    e = q[:1].expand(2, -1, -1, -1)
    both = ops.qk_norm_rope(e, e, q_weight=w, k_weight=w)
    assert torch.equal(both[0][0], both[0][1]) and torch.equal(both[0][0], want[0][0])
    odd = torch.randn((1, 2, 9, 65), generator=g).to(BF).cuda()[..., 1:]  # rows that are not aligned
    got = ops.qk_norm_rope(odd, odd, q_weight=w, k_weight=w)
    assert torch.equal(got[0], ops.qk_norm_rope(odd.contiguous(), odd.contiguous(), q_weight=w, k_weight=w)[0])


def test_constant_zero_and_non_finite_rows():
    """A layer norm of a constant row is its bias; zero rows stay zero; a row with NaN or inf spoils
    itself alone."""
    x = torch.randn((1, 2, 64, 64), generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    x[0, 0, 5] = 3.0
    x[0, 1, 6] = 0.0
    w = torch.full((64,), 2.0, device="cuda")
    b = torch.full((64,), 0.5, device="cuda")
    y = ops.qk_norm_rope(x, x, norm="layer", q_weight=w, k_weight=w, q_bias=b, k_bias=b)[0]
    assert (y[0, 0, 5] == 0.5).all() and (y[0, 1, 6] == 0.5).all()
    z = x.clone()
    z[0, 0, 7, 3], z[0, 1, 9, 0] = float("nan"), float("inf")
    bad = torch.zeros((1, 2, 64), dtype=torch.bool, device="cuda")
    bad[0, 0, 7] = bad[0, 1, 9] = True
    for norm in ("rms", "layer"):
        a, c = (ops.qk_norm_rope(t, t, norm=norm, q_weight=w, k_weight=w)[0] for t in (x, z))
        assert torch.equal(a[~bad], c[~bad]) and c[0, 0, 7].isnan().all()
    # eps = 0: rows past the last (a wave holds 4 or 8) add nothing to the weights' gradient
    for nhd in (False, True):
        q = torch.ones((1, 3, 5, 64) if not nhd else (1, 5, 3, 64), dtype=BF, device="cuda")
        q = q.transpose(1, 2) if nhd else q
        got = ops.qk_norm_rope_bwd(q, q, q, q, eps=0.0, q_weight=w, k_weight=w)
        assert (got[2] == 15).all() and (got[3] == 15).all()


@pytest.mark.parametrize("shape", [(0, 2, 8, 64), (1, 0, 8, 64), (1, 2, 0, 64)])
def test_empty_calls(shape):
    x = torch.empty(shape, dtype=BF, device="cuda")
    w = torch.ones(64, device="cuda")
    assert ops.qk_norm_rope(x, x, q_weight=w, k_weight=w)[0].shape == shape
    got = ops.qk_norm_rope_bwd(x, x, x, x, q_weight=w, k_weight=w)
    assert got[0].shape == shape and (got[2] == 0).all() and (got[3] == 0).all() and got[4] is None


def test_replays_in_a_graph_and_on_a_stream():
    q, k, kw = _setup(1, 6, 300, 300, 128, BF, True, "rms", False, "interleaved", 0, 300, "w", BF)
    run = lambda: (*ops.qk_norm_rope(q, k, **kw), *ops.qk_norm_rope_bwd(q, k, q, k, **kw)[:4])  # noqa: E731
    want = [t.clone() for t in run()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = run()
    for i in range(3):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        ops.qk_norm_rope(k, q, **kw)


def test_autograd():
    """The differentiable form is the two calls, weights' gradients in the weights' dtype; an unused
    output's gradient is zero."""
    q, k, kw = _setup(1, 3, 50, 50, 64, BF, True, "layer", False, "interleaved", 0, 50, "wb", BF)
    names = ("q_weight", "k_weight", "q_bias", "k_bias")
    leaves = [q.detach().requires_grad_(), k.detach().requires_grad_()] + [kw[n].detach().requires_grad_() for n in names]
    args = dict(kw, **dict(zip(names, leaves[2:])))
    y = md.qk_norm_rope(leaves[0], leaves[1], **args)
    dq, dk = torch.randn_like(q), torch.randn_like(k)
    got = torch.autograd.grad(y, leaves, (dq, dk))
    want = ops.qk_norm_rope_bwd(q, k, dq, dk, **kw)
    for a, c, leaf in zip(got, want, leaves):
        assert a.dtype == leaf.dtype and torch.equal(a, c.to(leaf.dtype))
    y = md.qk_norm_rope(leaves[0], leaves[1], **args)
    got = torch.autograd.grad(y[0], leaves, dq)
    assert torch.equal(got[0], want[0]) and (got[1] == 0).all() and (got[3] == 0).all()


def test_refusals():
    q, k, kw = _setup(1, 2, 16, 16, 64, BF, False, "rms", False, "interleaved", 0, 16, "w", BF)
    cases = [
        (ValueError, "differ in S", dict(k=k[:, :1])),
        (ValueError, "same dtype", dict(k=k.half())),
        (TypeError, "float16 or bfloat16", dict(q=q.float(), k=k.float())),
        (ValueError, "head_dim", dict(q=q[..., :32], k=k[..., :32])),
        (ValueError, "norm must be", dict(norm="batch")),
        (ValueError, "need a norm", dict(norm="none")),
        (ValueError, "eps", dict(eps=float("inf"))),
        (ValueError, "shape", dict(q_weight=kw["q_weight"][:32])),
        (TypeError, "share one", dict(q_weight=kw["q_weight"].float())),
        (TypeError, "share one", dict(q_weight=kw["q_weight"].double(), k_weight=kw["k_weight"].double())),
        (ValueError, "come together", dict(cos=None)),
        (TypeError, "float32", dict(cos=kw["cos"].double(), sin=kw["sin"].double())),
        (ValueError, "cos and sin must have shape", dict(cos=kw["cos"][:, :48], sin=kw["sin"][:, :48])),
        (ValueError, "exceed", dict(rope_offset=1)),
        (ValueError, "exceed", dict(rope_offset=-1)),
        (ValueError, "GPU", dict(q_weight=kw["q_weight"].cpu())),
        (ValueError, "out must be", dict(out=(q, k[:, :1]))),
        (ValueError, "apart", dict(out=(k, q))),
        (ValueError, "apart", dict(out=(q, q))),
        (ValueError, "apart", dict(out=(q, torch.empty_like(k[:, :1]).expand(-1, 2, -1, -1)))),
        (ValueError, "apart", dict(k=q, out=(q, k.clone()))),
        (ValueError, "apart", dict(out=(q.view(1, 16, 2, 64).transpose(1, 2), k))),
        (ValueError, "unit dim stride", dict(out=(q.transpose(2, 3).contiguous().transpose(2, 3), k.clone()))),
    ]
    for error, word, change in cases:
        a = dict(kw, q=q, k=k)
        a.update(change)
        with pytest.raises(error, match=word):
            ops.qk_norm_rope(**a)
    with pytest.raises(ValueError, match="grad_q"):
        ops.qk_norm_rope_bwd(q, k, q[:, :, :8], k, **kw)
    wide = torch.zeros((1, 65, 2, 128), dtype=BF, device="cuda")
    with pytest.raises(ValueError, match="8192"):
        ops.qk_norm_rope(wide, wide, across_heads=True)
