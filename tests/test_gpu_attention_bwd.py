"""Gradients of dense and block-sparse attention (GPU) against the formulas in 64 bits.

Tolerances, element by element. u = half a step of the storage type (2^-8 bf16, 2^-11 fp16). out is
the 64-bit output rounded to it, lse the 64-bit one rounded to fp32. With
A_ij = sum_d |dO_id| |V_jd| and C_i = sum_d |dO_id| |O_id|:
  P:     rounded for dV's product: u P; fp32 scores of a few units and the LSE: 2^-14 P
  delta: out's rounding, u C_i, and fp32 sums, 2^-17 C_i;  dP: 2^-17 A_ij
  dS:    (u + 2^-14) |dS| + P (u C_i + 2^-17 (A_ij + C_i))
  dV:    sum_i (u + 2^-14 + 2^-17) P_ij |dO_i| + u |dV|
  dQ:    scale sum_j (err dS_ij + 2^-17 |dS_ij|) |K_j| + u |dQ|, and dK likewise
where 2^-17 stands for fp32 sums (at most 128 f of their absolute terms), and 2^-25 for half the
step below fp16's normal range.
"""
import pytest
import torch

import mod_dit_amd as md
from mod_dit_amd import ops

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _tensors(B, H, Sq, Skv, D, dtype, nhd, seed=0, qscale=1.0, gscale=1.0):
    g = torch.Generator().manual_seed(seed)

    def one(S, scale=1.0):
        t = (torch.randn((B, S, H, D) if nhd else (B, H, S, D), generator=g) * scale).to(dtype).cuda()
        return t.transpose(1, 2) if nhd else t

    return one(Sq, qscale), one(Skv), one(Skv), one(Sq, gscale)


def _ref(q, k, v, do, scale, mask=None, dlse=None, u_out=None):
    """out, lse, gradients in 64 bits, and the gradients' tolerances (u |x| aside)."""
    u = torch.finfo(q.dtype).eps / 2
    u_out = u if u_out is None else u_out
    q, k, v, do = (t.double() for t in (q, k, v, do))
    s = q @ k.transpose(2, 3) * scale
    if mask is not None:
        s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None]).nan_to_num(0.0)
    out = p @ v
    dp = do @ v.transpose(2, 3)
    delta = (do * out).sum(-1, keepdim=True)
    if dlse is not None:
        delta = delta - dlse.double()[..., None]
    ds = p * (dp - delta)
    grads = (scale * ds @ k, scale * ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do)
    A, C = do.abs() @ v.abs().transpose(2, 3), (do.abs() * out.abs()).sum(-1, keepdim=True)
    if dlse is not None:
        C = C + dlse.double().abs()[..., None]
    err = (u + 2.0 ** -14 + 2.0 ** -17) * ds.abs() + p * (u_out * C + 2.0 ** -17 * (A + C))
    tol = (scale * err @ k.abs(), scale * err.transpose(2, 3) @ q.abs(),
           (u + 2.0 ** -14 + 2.0 ** -17) * p.transpose(2, 3) @ do.abs())
    return out, lse, grads, tol


def _check(got, grads, tol, dtype):
    u = torch.finfo(dtype).eps / 2
    for name, a, w, t in zip(("dq", "dk", "dv"), got, grads, tol):
        lim = t + u * w.abs() + 2.0 ** -25
        off = (a.double() - w).abs()
        assert a.dtype == dtype and a.shape == w.shape
        assert (off <= lim).all(), (name, (off / lim).max().item())


def _run(q, k, v, do, scale=None, mask=None, tiles=None, dlse=None, **kw):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse, grads, tol = _ref(q, k, v, do, scale, mask, dlse)
    out, lse = out.to(q.dtype), lse.float()
    if tiles is None:
        call = lambda: ops.flash_bwd(q, k, v, out, lse, do, scale, dlse)  # noqa: E731
    else:
        call = lambda: ops.block_sparse_bwd(q, k, v, out, lse, do, tiles, scale, dlse, **kw)  # noqa: E731
    got = call()
    _check(got, grads, tol, q.dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, call()))
    return got


@pytest.mark.parametrize("B,H,Sq,Skv,D,dtype,nhd", [
    (1, 1, 1, 1, 64, BF, False),
    (1, 2, 1, 1, 128, FP, True),
    (1, 1, 2, 63, 128, BF, False),
    (2, 1, 63, 2, 64, FP, True),
    (1, 3, 64, 64, 128, BF, True),
    (2, 2, 65, 65, 64, BF, False),
    (1, 2, 127, 129, 128, FP, True),
    (2, 3, 129, 127, 64, FP, False),
    (1, 2, 1, 700, 128, BF, True),
    (1, 2, 700, 1, 64, BF, False),
    (1, 2, 391, 640, 128, BF, False),
    (1, 2, 640, 391, 128, FP, True),
    (1, 5, 1577, 1577, 64, BF, True),
    (1, 2, 2100, 2100, 128, FP, False),
])
def test_dense(B, H, Sq, Skv, D, dtype, nhd):
    _run(*_tensors(B, H, Sq, Skv, D, dtype, nhd))


def _token_mask(m, tiles_union, block, S, origin):
    """Executed token mask (1,H,S,S) of a block mask: 64-row halves, or pairs where rows are united."""
    nb = m.shape[1]
    if tiles_union and block == 64:
        pair = torch.arange(nb, device="cuda") // 2 * 2
        m = m[:, pair] | m[:, (pair + 1).clamp(max=nb - 1)]
    at = (torch.arange(S, device="cuda") - origin) // block
    return m[:, at][:, :, at][None]


SPARSE = [
    (2, 640, 64, BF, 64, 0, False, False),
    (3, 640, 128, FP, 64, 0, True, True),
    (2, 677, 128, BF, 64, -27, False, True),
    (1, 700, 64, FP, 64, -63, True, False),
    (2, 1024, 128, BF, 128, 0, True, False),
    (2, 833, 64, BF, 128, -1, False, False),
    (1, 130, 128, BF, 64, 0, False, False),
    (2, 64, 64, FP, 64, 0, True, False),
    (1, 2112, 128, BF, 64, 0, False, True),
]


@pytest.mark.parametrize("H,S,D,dtype,block,origin,union,nhd", SPARSE)
def test_sparse(H, S, D, dtype, block, origin, union, nhd):
    """Random masks with empty rows and key columns that nobody attends to."""
    g = torch.Generator().manual_seed(3)
    nb = -(-(S - origin) // block)
    m = torch.rand((H, nb, nb), generator=g) < 0.4
    if nb > 2:
        m[:, nb // 2:nb // 2 + 2] = False
        m[:, :, 1] = False
    m = m.cuda()
    tiles = ops.mask_to_tiles(m, block, union_rows=union, grid_origin=origin)
    q, k, v, do = _tensors(1, H, S, S, D, dtype, nhd)
    mask = _token_mask(m, union, block, S, origin)
    got = _run(q, k, v, do, mask=mask, tiles=tiles)
    kept = _run(q, k, v, do, mask=mask, tiles=tiles, key_tiles=ops.transpose_tiles(tiles, S))
    assert all(torch.equal(a, b) for a, b in zip(got, kept))
    assert (got[0][~mask.any(-1)] == 0).all()
    dead = ~mask.any(-2)
    assert (got[1][dead] == 0).all() and (got[2][dead] == 0).all()


def test_sparse_with_more_queries_than_keys_and_batch():
    """The video rows of a padded layout: a prefix of the queries against all valid keys."""
    g = torch.Generator().manual_seed(4)
    m = (torch.rand((2, 6, 9), generator=g) < 0.5).cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    q, k, v, do = _tensors(2, 2, 384, 550, 64, BF, True)
    mask = m.repeat_interleave(64, 1).repeat_interleave(64, 2)[None, :, :, :550].expand(2, -1, -1, -1)
    _run(q, k, v, do, mask=mask, tiles=tiles)


@pytest.mark.parametrize("D,dtype", [(64, FP), (128, BF)])
@pytest.mark.parametrize("rows,keys", [(190, 70 * 640), (70 * 640, 150)])
def test_lists_of_many_entries(D, dtype, rows, keys):
    """Lists longer than a workgroup arranges at a time, most of their entries for one half alone."""
    g = torch.Generator().manual_seed(6)
    m = (torch.rand((1, -(-rows // 64), -(-keys // 64)), generator=g) < 0.6).cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    q, k, v, do = _tensors(1, 1, rows, keys, D, dtype, False)
    mask = m.repeat_interleave(64, 1).repeat_interleave(64, 2)[None, :, :rows, :keys]
    _run(q, k, v, do, mask=mask, tiles=tiles)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, FP)])
@pytest.mark.parametrize("rows,keys,batch", [(190, 70 * 640, 24), (70 * 640, 150, 40)])
def test_lists_of_many_entries_on_a_full_card(D, dtype, rows, keys, batch):
    """The same with so many workgroups that none shares its list: every batch has the first's result."""
    g = torch.Generator().manual_seed(6)
    m = (torch.rand((1, -(-rows // 64), -(-keys // 64)), generator=g) < 0.6).cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    q, k, v, do = _tensors(1, 1, rows, keys, D, dtype, False)
    mask = m.repeat_interleave(64, 1).repeat_interleave(64, 2)[None, :, :rows, :keys]
    out, lse, grads, tol = _ref(q, k, v, do, D ** -0.5, mask)
    many = [t.expand(batch, *t.shape[1:]) for t in (q, k, v, out.to(dtype), lse.float(), do)]
    got = ops.block_sparse_bwd(*many, tiles)
    _check([t[:1] for t in got], grads, tol, dtype)
    assert all(torch.equal(t, t[:1].expand_as(t)) for t in got)


@pytest.mark.parametrize("H,nq,nk,p", [(1, 1, 1, 1.0), (2, 5, 3, 0.5), (3, 40, 70, 0.1), (1, 7, 33, 0.0), (2, 130, 64, 0.9)])
def test_transpose_tiles(H, nq, nk, p):
    """Every (query block, key tile) pair of the lists, and no other, in ascending order."""
    g = torch.Generator().manual_seed(5)
    m = (torch.rand((H, 2 * nq, nk), generator=g) < p).cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    got = ops.transpose_tiles(tiles, nk * 64)
    assert got.n_ktiles == (nk + 1) // 2 and got.cap == 4 * nq // 2
    pad = torch.cat([m, m.new_zeros((H, 2 * nq, nk % 2))], 2).cpu()
    for h in range(H):
        for t in range(got.n_ktiles):
            bits = pad[h, :, 2 * t].int() + 2 * pad[h, :, 2 * t + 1].int()
            want = [(i << 2) | b for i, b in enumerate(bits.tolist()) if b]
            n = got.counts[h, t].item()
            assert got.entries[h, t, :n].tolist() == want


def test_a_large_layer():
    """A HunyuanVideo-like layer, 24 heads of 115,163 tokens, 17 % of the blocks: sampled rows of dQ and
    of dK and dV. out and lse are the forward's own, so that their rounding is part of the formula."""
    H, S, D, scale, u = 24, 115163, 128, 128 ** -0.5, 2.0 ** -8
    g = torch.Generator("cuda").manual_seed(7)
    q, k, v, do = (torch.randn((1, S, H, D), generator=g, device="cuda").to(BF).transpose(1, 2) for _ in range(4))
    m = torch.rand((H, 1800, 1800), generator=g, device="cuda") < 0.17
    m[:, :, 700] = True
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    out, lse = ops.block_sparse_fwd(q, k, v, tiles, return_lse=True)
    got = ops.block_sparse_bwd(q, k, v, out, lse, do, tiles)
    for h in (0, 11, 23):
        Q, K, V, dO, L = (t[0, h].double() for t in (q, k, v, do, lse))
        C = (dO * out[0, h].double()).abs().sum(-1)
        delta = (dO * out[0, h].double()).sum(-1)
        pick = torch.tensor([0, 63, 64, 127, 44800, 44863, 60001, 115100, S - 1], device="cuda")
        allowed = m[h][pick // 64].repeat_interleave(64, 1)[:, :S]
        p = torch.exp(Q[pick] @ K.T * scale - L[pick, None]).masked_fill(~allowed, 0.0)
        ds = p * (dO[pick] @ V.T - delta[pick, None])
        err = (u + 2.0 ** -14 + 2.0 ** -17) * ds.abs() + p * 2.0 ** -17 * (dO[pick].abs() @ V.abs().T + C[pick, None])
        want, tol = scale * ds @ K, scale * err @ K.abs()
        assert ((got[0][0, h, pick].double() - want).abs() <= tol + u * want.abs() + 2.0 ** -25).all()
        allowed = m[h][:, pick // 64].repeat_interleave(64, 0)[:S]
        p = torch.exp(Q @ K[pick].T * scale - L[:, None]).masked_fill(~allowed, 0.0)
        ds = p * (dO @ V[pick].T - delta[:, None])
        err = (u + 2.0 ** -14 + 2.0 ** -17) * ds.abs() + p * 2.0 ** -17 * (dO.abs() @ V[pick].abs().T + C[:, None])
        want, tol = scale * ds.T @ Q, scale * err.T @ Q.abs()
        assert ((got[1][0, h, pick].double() - want).abs() <= tol + u * want.abs() + 2.0 ** -25).all()
        want, tol = p.T @ dO, (u + 2.0 ** -14 + 2.0 ** -17) * p.T @ dO.abs()
        assert ((got[2][0, h, pick].double() - want).abs() <= tol + u * want.abs() + 2.0 ** -25).all()


def test_entries_past_the_last_tile():
    """A 128-token mask whose last block the sequence half fills lists a key tile past the end."""
    m = torch.ones((1, 3, 3), dtype=torch.bool, device="cuda")
    tiles = ops.mask_to_tiles(m, 128, union_rows=False)
    q, k, v, do = _tensors(1, 1, 300, 300, 64, BF, False)
    got = _run(q, k, v, do, mask=torch.ones((1, 1, 300, 300), dtype=torch.bool, device="cuda"), tiles=tiles)
    out, lse = ops.flash_fwd(q, k, v)
    assert got[0].isfinite().all()


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, FP)])
def test_gradient_of_the_lse(D, dtype):
    q, k, v, do = _tensors(1, 2, 200, 260, D, dtype, False)
    dlse = torch.randn((1, 2, 200), generator=torch.Generator().manual_seed(6)).cuda()
    _run(q, k, v, do, dlse=dlse)
    _run(q, k, v, torch.zeros_like(do), dlse=dlse)


@pytest.mark.parametrize("gscale", [2.0 ** -12, 1.0, 2.0 ** 9])
def test_half_precision_gradients_of_any_size(gscale):
    """dS at fp16 holds its precision for small and loss-scaled gradients: outputs that do not
    leave fp16 themselves come back within the same relative tolerance. One long row of keys, so
    that P is far below fp16's smallest normal value."""
    q, k, v, do = _tensors(1, 1, 130, 4100, 64, FP, False, gscale=gscale)
    _run(q, k, v, do)


@pytest.mark.parametrize("qscale", [0.0, 8.0])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_flat_and_peaked_scores(qscale, dtype):
    """Equal scores, and scores of a deviation of 8 (fp32 rounds those to 2^-18: the 2^-14 of the
    tolerance holds up to 2^4 units times 16 terms' worth of rounding)."""
    _run(*_tensors(1, 2, 150, 300, 64, dtype, False, qscale=qscale))


@pytest.mark.parametrize("Skv", [2, 3, 17, 63, 64])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("with_dlse", [False, True])
def test_few_keys_do_not_see_the_rounding_of_out(Skv, D, with_dlse):
    """bf16 with up to 64 keys: delta is formed from P and dP, so that its error is that of fp32 sums
    (2^-14 P as in P itself), not that of out's rounding."""
    q, k, v, do = _tensors(1, 3, 200, Skv, D, BF, True, qscale=2.0)
    scale = D ** -0.5
    dlse = torch.randn((1, 3, 200), generator=torch.Generator().manual_seed(1)).cuda() if with_dlse else None
    out, lse, grads, tol = _ref(q, k, v, do, scale, None, dlse, u_out=2.0 ** -14)
    got = ops.flash_bwd(q, k, v, out.to(BF), lse.float(), do, scale, dlse)
    _check(got, grads, tol, BF)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sparse", [False, True])
def test_one_key(dtype, sparse):
    """The softmax of one key does not depend on q and k: their gradients are exactly zero, and with a
    gradient of the LSE its own."""
    q, k, v, do = _tensors(2, 2, 150, 1, 128, dtype, False)
    tiles = None
    if sparse:
        m = torch.ones((2, 3, 1), dtype=torch.bool, device="cuda")
        tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    got = _run(q, k, v, do, tiles=tiles)
    assert (got[0] == 0).all() and (got[1] == 0).all()
    dlse = torch.randn((2, 2, 150), generator=torch.Generator().manual_seed(1)).cuda()
    _run(q, k, v, do, tiles=tiles, dlse=dlse)


def test_non_finite_values_stay_where_no_pair_reaches():
    """NaN and inf in keys, values and gradients of tiles that the mask drops, and past the ends of
    strided slices, change nothing."""
    g = torch.Generator().manual_seed(7)
    m = torch.rand((2, 6, 6), generator=g) < 0.6
    m[:, 2], m[:, :, 4] = False, False
    m = m.cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    q, k, v, do = _tensors(1, 2, 384, 384, 128, BF, True)
    out, lse, *_ = _ref(q, k, v, do, 128 ** -0.5, _token_mask(m, False, 64, 384, 0))
    out, lse = out.to(BF), lse.float()
    want = ops.block_sparse_bwd(q, k, v, out, lse, do, tiles)
    for t, rows in ((q, slice(128, 192)), (do, slice(128, 192)), (k, slice(256, 320)), (v, slice(256, 320))):
        t[:, :, rows][:, :, ::2] = float("nan")
        t[:, :, rows][:, :, 1::2] = float("inf")
    got = ops.block_sparse_bwd(q, k, v, out, lse, do, tiles)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    long = [torch.full((1, 500, 2, 64), float("nan"), dtype=BF, device="cuda") for _ in range(5)]
    q, k, v, do = _tensors(1, 2, 300, 333, 64, BF, False)
    out, lse, *_ = _ref(q, k, v, do, 0.125)
    out, lse = out.to(BF), lse.float()
    want = ops.flash_bwd(q, k, v, out, lse, do)
    views = []
    for buf, t in zip(long, (q, k, v, out, do)):
        view = buf.transpose(1, 2)[:, :, 100:100 + t.shape[2]]
        view.copy_(t)
        views.append(view)
    got = ops.flash_bwd(*views[:4], lse, views[4])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_very_low_scores():
    """Scores near -300: the LSE is far below zero, where 2^-LSE alone would overflow."""
    q, k, v, do = _tensors(1, 1, 100, 70, 64, BF, False)
    q[..., 0], k[..., 0] = 50.0, -50.0
    _run(q, k, v, do)


def test_broadcast_keys_and_unaligned_rows():
    q, k, v, do = _tensors(2, 3, 100, 150, 64, BF, False)
    e = lambda t: t[:1, :1].expand(2, 3, -1, -1)  # noqa: E731
    _run(q, e(k), e(v), do)
    row = lambda t: t[:, :, :1].expand(-1, -1, 150, -1)  # noqa: E731
    _run(q, row(k), row(v), do)  # one row for every token: past the last it must not be read
    _run(row(q), k, v, row(do))
    odd = torch.randn((1, 2, 70, 65), generator=torch.Generator().manual_seed(1)).to(BF).cuda()[..., 1:]
    _run(odd, odd, odd, odd)


@pytest.mark.parametrize("Sq,Skv", [(0, 5), (5, 0), (0, 0)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_empty_sides(Sq, Skv, dtype):
    q, k, v, do = _tensors(1, 2, Sq, Skv, 64, dtype, False)
    lse = torch.full((1, 2, Sq), float("-inf"), device="cuda")
    for t in ops.flash_bwd(q, k, v, do, lse, do):
        assert (t == 0).all()
    nq, cap = (Sq + 127) // 128, (Skv + 63) // 64
    tiles = ops.TileList(torch.zeros((2, nq), dtype=torch.int32, device="cuda"),
                         torch.zeros((2, nq, cap), dtype=torch.int32, device="cuda"), 64, False)
    for t, x in zip(ops.block_sparse_bwd(q, k, v, do, lse, do, tiles), (q, k, v)):
        assert t.shape == x.shape and (t == 0).all()


def test_gradients_against_differences():
    """Along random directions, against central differences of the 64-bit loss; the tolerance adds
    the gradients' own."""
    q, k, v, do = _tensors(1, 2, 130, 200, 64, BF, False)
    out, lse, grads, tol = _ref(q, k, v, do, 0.125)
    got = ops.flash_bwd(q, k, v, out.to(BF), lse.float(), do)
    at = [t.double() for t in (q, k, v)]
    f = lambda q, k, v: (torch.softmax(q @ k.transpose(2, 3) * 0.125, -1) @ v * do.double()).sum()  # noqa: E731
    g = torch.Generator().manual_seed(8)
    for i in range(3):
        d = torch.randn(at[i].shape, generator=g, dtype=torch.float64).cuda()
        h = 1e-5
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + h * d, at[i] - h * d
        diff = ((f(*plus) - f(*minus)) / (2 * h)).item()
        lim = (d.abs() * (tol[i] + 2.0 ** -8 * grads[i].abs())).sum().item()
        assert abs((got[i].double() * d).sum().item() - diff) <= lim + 1e-6 * abs(diff) + 1e-6


def test_streams_and_graphs():
    q, k, v, do = _tensors(1, 2, 400, 400, 128, BF, True)
    m = (torch.rand((2, 7, 7), generator=torch.Generator().manual_seed(2)) < 0.5).cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False)
    out, lse = ops.block_sparse_fwd(q, k, v, tiles, return_lse=True)
    run = lambda: ops.block_sparse_bwd(q, k, v, out, lse, do, tiles)  # noqa: E731
    want = [t.clone() for t in run()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for i in range(3):
        for g, got in zip(graphs, outs):
            for t in got:
                t.zero_()
            g.replay()
        torch.cuda.synchronize()
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        ops.flash_bwd(q, k, v, out, lse, do)


def _layer(B, H, S, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn((B, S, H, D), generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(3))
    w = [(torch.rand(D, generator=g) + 0.5).cuda() for _ in range(2)]
    a = torch.rand((S, D // 2), generator=g) * 6.28
    return q, k, v, w, a.cos().cuda(), a.sin().cuda()


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_a_training_step_of_a_layer(sparse, dtype):
    """Norm and rotation, attention and their gradients by autograd: the same as the calls one after
    the other, each of which is checked against 64 bits above."""
    B, H, S, D = 2, 2, 330, 64
    q, k, v, w, cos, sin = _layer(B, H, S, D, dtype)
    m = (torch.rand((H, 6, 6), generator=torch.Generator().manual_seed(1)) < 0.5).cuda()
    tiles = ops.mask_to_tiles(m, 64, union_rows=False) if sparse else None
    leaves = [t.detach().requires_grad_() for t in (q, k, v, *w)]
    kw = dict(cos=cos, sin=sin)
    a, b = md.qk_norm_rope(leaves[0], leaves[1], q_weight=leaves[3], k_weight=leaves[4], **kw)
    if sparse:
        y, lse = md.block_sparse_attention(a, b, leaves[2], tiles, return_lse=True)
    else:
        y, lse = md.flash_attention(a, b, leaves[2], return_lse=True)
    dy = torch.randn_like(y)
    dl = torch.zeros_like(lse).masked_fill(lse.isfinite(), 0.01)
    got = torch.autograd.grad((y, lse), leaves, (dy, dl))
    kw.update(q_weight=w[0], k_weight=w[1])
    a, b = ops.qk_norm_rope(q, k, **kw)
    fwd = (lambda: ops.block_sparse_fwd(a, b, v, tiles, return_lse=True)) if sparse else (lambda: ops.flash_fwd(a, b, v))
    out, l2 = fwd()
    assert torch.equal(out, y) and torch.equal(l2, lse)
    if sparse:
        da, db, dv = ops.block_sparse_bwd(a, b, v, out, lse, dy, tiles, grad_lse=dl)
    else:
        da, db, dv = ops.flash_bwd(a, b, v, out, lse, dy, grad_lse=dl)
    dq, dk, dwq, dwk, _, _ = ops.qk_norm_rope_bwd(q, k, da, db, **kw)
    for x, want in zip(got, (dq, dk, dv, dwq, dwk)):
        assert torch.equal(x, want)


def test_a_training_step_in_a_graph():
    """Forward and backward of a layer on leaves of their own, captured and replayed."""
    q, k, v, w, cos, sin = _layer(1, 2, 200, 64, BF, 3)
    dy = torch.randn_like(q)

    def step():
        leaves = [t.detach().requires_grad_() for t in (q, k, v, *w)]
        a, b = md.qk_norm_rope(leaves[0], leaves[1], q_weight=leaves[3], k_weight=leaves[4], cos=cos, sin=sin)
        return torch.autograd.grad(md.flash_attention(a, b, leaves[2]), leaves, dy)

    want = [t.clone() for t in step()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(3):
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_autograd_edges():
    q, k, v, do = _tensors(1, 2, 90, 90, 64, BF, False)
    a, b, c = (t.detach().requires_grad_() for t in (q, k, v))
    y, lse = md.flash_attention(a, b, c, return_lse=True)
    assert y.requires_grad and lse.requires_grad
    only = torch.autograd.grad(lse.sum(), (a, b, c))
    assert (only[2] == 0).all()  # the LSE does not see the values
    y = md.flash_attention(q, k, c)  # one leaf
    assert torch.equal(torch.autograd.grad(y, c, do)[0], ops.flash_bwd(q, k, v, y.detach(), lse.detach(), do)[2])
    assert not md.flash_attention(q, k, v).requires_grad
    shared = k[:, :1].detach().requires_grad_()  # one head's keys for both
    y = md.flash_attention(q, shared.expand(-1, 2, -1, -1), v)
    g = torch.autograd.grad(y, shared, do)[0]
    assert g.shape == shared.shape and g.isfinite().all()
    x = a * 1.0
    y = md.flash_attention(x, b, c)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        torch.autograd.grad(torch.autograd.grad(y, a, do, create_graph=True)[0].sum(), a)


def test_refusals():
    q, k, v, do = _tensors(1, 2, 100, 100, 64, BF, False)
    out, lse = ops.flash_fwd(q, k, v)
    tiles = ops.mask_to_tiles(torch.ones((2, 2, 2), dtype=torch.bool, device="cuda"), 64)
    other = ops.mask_to_tiles(torch.ones((3, 2, 2), dtype=torch.bool, device="cuda"), 64)
    cases = [
        (ValueError, "incompatible", dict(v=v[:, :, :50])),
        (ValueError, "out and grad_out", dict(grad_out=do[:, :, :50])),
        (ValueError, "same dtype", dict(grad_out=do.half())),
        (TypeError, "float16 or bfloat16", {n: t.float() for n, t in dict(q=q, k=k, v=v, out=out, grad_out=do).items()}),
        (ValueError, "lse must be", dict(lse=lse.double())),
        (ValueError, "lse must be", dict(lse=lse[:, :, :50])),
        (ValueError, "grad_lse must be", dict(grad_lse=lse[:, :1])),
        (ValueError, "GPU", dict(lse=lse.cpu())),
    ]
    for error, word, change in cases:
        a = dict(q=q, k=k, v=v, out=out, lse=lse, grad_out=do)
        a.update(change)
        with pytest.raises(error, match=word):
            ops.flash_bwd(**a)
        with pytest.raises(error, match=word):
            ops.block_sparse_bwd(**a, tiles=tiles)
    with pytest.raises(ValueError, match="heads"):
        ops.block_sparse_bwd(q, k, v, out, lse, do, other)
    with pytest.raises(ValueError, match="transposed"):
        ops.block_sparse_bwd(q, k, v, out, lse, do, tiles, key_tiles=ops.transpose_tiles(other, 100))
    with pytest.raises(ValueError, match="tile lists"):
        bad = ops.TileList(tiles.counts.long(), tiles.entries, 64, True)
        ops.block_sparse_bwd(q, k, v, out, lse, do, bad)
    short = ops.mask_to_tiles(torch.ones((2, 1, 2), dtype=torch.bool, device="cuda"), 64)
    with pytest.raises(md._lib.ModditError, match="n_qtiles|needs"):
        long = _tensors(1, 2, 300, 100, 64, BF, False)
        ops.block_sparse_bwd(long[0], long[1], long[2], long[3], torch.zeros((1, 2, 300), device="cuda"), long[3], short)
