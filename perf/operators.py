"""Performance cases of the training-side operators: the per-head norm of queries and keys
with their position rotation, its gradient, and the gradients of dense and block-sparse
attention.

`listed()` names the cases, `draw(rng)` gives others of the same ranges, `prepare` makes what a
program holds before the call, `run` is one call, `exact` the same result in 64 bits. With
`own` false `run` computes the operators from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = 10.0 * 12 * 29019.0**2 * 128  # FLOP of the largest listed case


def _norm(op, heads, tokens, dim, **kw):
    """op: 'rotate' (norm and rotation of q and k), 'rotate-grad' (its gradients)."""
    c = dict(op=op, batch=1, heads=heads, tokens=tokens, dim=dim, dtype="bf16", storage="nhd",
             norm="rms", across=False, offset=0, rotated=tokens, pairs="interleaved")
    c.update(kw)
    return c


def _grad(op, heads, rows, keys, dim, **kw):
    """op: 'dense-grad', 'sparse-grad' (64x64 blocks, `keep` of them), 'layer' (norm and
    rotation, block-sparse attention, and the gradients of both)."""
    c = dict(op=op, batch=1, heads=heads, rows=rows, keys=keys, dim=dim, dtype="bf16",
             storage="nhd", keep=0.0, origin=0, union=False)
    c.update(kw)
    return c


def listed():
    return [
        # one token of a layer: the call's own latency
        dict(_norm("rotate", 24, 1, 128), name="rotate-1"),
        # the HunyuanVideo-like headline layer: RMS norms per head, every video token rotated
        dict(_norm("rotate", 24, 115200, 128), name="rotate-hunyuan-115k"),
        # the Wan-like layer: one RMS norm over all of a token's heads
        dict(_norm("rotate", 40, 69120, 128, across=True), name="rotate-wan-69k"),
        # training a CogVideoX-like layer: layer norm per head, text first and not rotated
        dict(_norm("rotate-grad", 48, 17776, 64, dtype="fp16", norm="layer", storage="hnd",
                   offset=226, rotated=17550), name="rotate-grad-cogvideox-17k"),
        # training a Wan-like layer on a shorter clip
        dict(_norm("rotate-grad", 40, 28800, 128, across=True), name="rotate-grad-wan-29k"),
        # attention gradients of the smallest layer in use: 4 frames x 32x32 tokens, 2 heads
        dict(_grad("dense-grad", 2, 4096, 4096, 64, dtype="fp16"), name="dense-grad-plumbing-4k"),
        # one latent frame (an image) of a CogVideoX-like layer, odd length
        dict(_grad("dense-grad", 48, 1577, 1577, 64, storage="hnd"), name="dense-grad-image-1577"),
        # a HunyuanVideo-like clip with its valid text tokens, half of the layer's heads
        dict(_grad("dense-grad", 12, 29019, 29019, 128), name="dense-grad-hunyuan-29k"),
        # the text rows of that layer against all of its keys
        dict(_grad("dense-grad", 24, 256, 29019, 128), name="dense-grad-text-256"),
        # fine-tuning that clip's layer under a predicted mask, 64x64 blocks kept exact
        dict(_grad("sparse-grad", 12, 28800, 28800, 128, keep=0.19), name="sparse-grad-hunyuan-29k"),
        # a CogVideoX-like layer on its shifted grid (226 text tokens first), a third of the heads
        dict(_grad("sparse-grad", 16, 17776, 17776, 64, dtype="fp16", keep=0.35, origin=-30),
             name="sparse-grad-cogvideox-17k"),
        # a whole training step of a short layer: norm, rotation, sparse attention and back
        dict(_grad("layer", 12, 7680, 7680, 128, keep=0.3), name="layer-7680"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the same kinds: one token to 115k for the norms, 1 to 29k rows and keys for
    the gradients of attention, 1 to 48 heads, both head dims and data types."""
    op = rng.choice(["rotate", "rotate-grad", "dense-grad", "dense-grad", "sparse-grad", "sparse-grad",
                     "layer"])
    dim = rng.choice([64, 128])
    kw = dict(dtype=rng.choice(["bf16", "bf16", "fp16"]), storage=rng.choice(["nhd", "hnd"]))
    if op.startswith("rotate"):
        tokens = _log_int(rng, 1, 115200)
        heads = max(1, min(_log_int(rng, 1, 48), int(24 * 115200 * 128 / (tokens * dim))))
        norm = rng.choice(["rms", "rms", "layer", "none"])
        offset = rng.choice([0, min(tokens - 1, 226), rng.randint(0, tokens - 1)])
        rotated = rng.choice([tokens - offset, rng.randint(1 if norm == "none" else 0, tokens - offset)])
        return _norm(op, heads, tokens, dim, norm=norm, across=rng.choice([False, False, True]),
                     offset=offset, rotated=rotated,
                     pairs=rng.choice(["interleaved", "interleaved", "halves"]),
                     batch=rng.choice([1, 1, 2]) if tokens * heads * dim < 24 * 57600 * 128 else 1, **kw)
    rows = _log_int(rng, 1 if op == "dense-grad" else 512, 29019 if op != "layer" else 8192)
    keys = rng.choice([rows, _log_int(rng, 1, 29019)]) if op == "dense-grad" else rows
    heads = max(1, min(_log_int(rng, 1, 48), int(LARGEST / (10.0 * rows * keys * 128))))
    if op != "dense-grad":
        kw.update(keep=round(rng.uniform(0.05, 0.7), 3), origin=rng.choice([0, -rng.randint(1, 63)]),
                  union=rng.choice([False, True]))
    return _grad(op, heads, rows, keys, dim, **kw)


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------
def _tensor(c, tokens, g, scale=1.0):
    """(B,H,tokens,D) normal values, stored as the case's projections are."""
    B, H, D = c["batch"], c["heads"], c["dim"]
    shape = (B, tokens, H, D) if c["storage"] == "nhd" else (B, H, tokens, D)
    t = (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[c["dtype"]])
    return t.transpose(1, 2) if c["storage"] == "nhd" else t


def _like(c, x):
    """x (B,H,tokens,D) in the case's type and storage."""
    x = x.to(DTYPES[c["dtype"]])
    if c["storage"] == "nhd":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    return x.contiguous()


def _tables(tokens, dim, pairs):
    """(cos, sin) of the positions 0.. : (tokens, D), each value at both elements of an
    interleaved pair, or (tokens, D/2) for pairs of halves."""
    pos = torch.arange(tokens, device="cuda", dtype=torch.float64)[:, None]
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    a = pos * inv
    if pairs == "interleaved":
        a = a.repeat_interleave(2, dim=-1)
    return a.cos().float(), a.sin().float()


def _norm_state(c, tokens, g):
    s = {"wq": None, "wk": None, "bq": None, "bk": None, "cos": None, "sin": None}
    n = c["dim"] * (c["heads"] if c["across"] else 1)
    dt = DTYPES[c["dtype"]]
    if c["norm"] != "none":
        s["wq"], s["wk"] = (torch.empty(n, device="cuda").normal_(1.0, 0.2, generator=g).to(dt) for _ in "qk")
    if c["norm"] == "layer":
        s["bq"], s["bk"] = (torch.empty(n, device="cuda").normal_(0.0, 0.1, generator=g).to(dt) for _ in "qk")
    if c["rotated"]:
        s["cos"], s["sin"] = _tables(c["rotated"], c["dim"], c["pairs"])
    return s


def _attention_inputs(c, g):
    """Queries and keys after norm and rotation: unit noise plus, per head, features shared by
    tokens that lie near each other, at a strength of its own."""
    def features(tokens):
        t = torch.arange(tokens, device="cuda", dtype=torch.float32)[:, None] / 64.0
        a = t * w  # (H, tokens, 16)
        return torch.cat([a.cos(), a.sin()], dim=-1) * strength

    B, H, D = c["batch"], c["heads"], c["dim"]
    w = torch.randn((H, 1, 16), generator=g, device="cuda") * 0.3
    strength = 0.3 + 1.2 * torch.rand((H, 1, 1), generator=g, device="cuda")
    q, k = (torch.randn((B, H, n, D), generator=g, device="cuda") for n in (c["rows"], c["keys"]))
    q[..., :32] += features(c["rows"])
    k[..., :32] += features(c["keys"])
    v = _tensor(c, c["keys"], g)
    # gradients of a loss that is averaged over the batch in bf16, and scaled up in fp16
    do = _tensor(c, c["rows"], g, scale=1e-3 if c["dtype"] == "bf16" else 1.0)
    return _like(c, q), _like(c, k), v, do


def _blocks(c, g):
    """Bool (H, n, n) 64x64 blocks: near ones, stripes and single columns, `keep` of all; the
    middle row of blocks of each head's last third is empty."""
    H, n = c["heads"], -(-(c["rows"] - c["origin"]) // 64)
    i = torch.arange(n, device="cuda")
    d = i[:, None] - i[None, :]
    score = torch.rand((H, n, n), generator=g, device="cuda") + torch.exp(-d.abs() / (0.05 * n + 1.0))
    score += 0.6 * (torch.rand((H, 1, n), generator=g, device="cuda") < 0.1)
    score += 0.6 * (torch.rand((H, 2 * n - 1), generator=g, device="cuda") < 0.1)[:, d + n - 1]
    k = max(1, int(round(c["keep"] * n * n)))
    m = score >= score.flatten(1).topk(k, dim=1).values[:, -1, None, None]
    m[2 * H // 3:, n // 2] = False
    if c["union"]:
        pair = i // 2 * 2
        m = m[:, pair] | m[:, (pair + 1).clamp(max=n - 1)]
    return m


def _lists(m):
    """counts (H, pairs of block rows) and entries of the active key tiles, ascending:
    (key tile << 2) | bit 0 for the pair's first block row | bit 1 for its second."""
    H, n, cols = m.shape
    if n % 2:
        m = torch.cat([m, m.new_zeros((H, 1, cols))], dim=1)
    bits = m[:, 0::2].int() | (m[:, 1::2].int() << 1)
    at = torch.arange(cols, device=m.device, dtype=torch.int32)
    key = torch.where(bits > 0, at, at + cols)
    order = key.sort(dim=-1).indices
    entries = ((at << 2) | bits).gather(2, order)
    return (bits > 0).sum(dim=-1, dtype=torch.int32), entries.contiguous()


def _token_mask(c, blocks, h=slice(None)):
    at = (torch.arange(c["rows"], device="cuda") - c["origin"]) // 64
    return blocks[h][:, at][:, :, at]


def _forward(c, s):
    """out (storage type) and natural-log LSE of the attention whose gradients a case asks for."""
    out = torch.empty(s["q"].shape, device="cuda")
    lse = torch.empty(s["q"].shape[:3], device="cuda")
    for b in range(c["batch"]):
        for h in range(c["heads"]):
            x = s["q"][b, h].float() @ s["k"][b, h].float().T * c["dim"] ** -0.5
            if "blocks" in s:
                x.masked_fill_(~_token_mask(c, s["blocks"], slice(h, h + 1))[0], float("-inf"))
            lse[b, h] = torch.logsumexp(x, dim=-1)
            out[b, h] = x.sub_(lse[b, h][:, None]).exp_().nan_to_num_(0.0) @ s["v"][b, h].float()
    return _like(c, out), lse


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"c": c}
    if c["op"].startswith("rotate"):
        s.update(_norm_state(c, c["tokens"], g))
        # projections whose channels differ in size
        s["q"], s["k"] = (_tensor(c, c["tokens"], g, scale=2.0 * torch.rand(c["dim"], generator=g, device="cuda")
                                  + 0.2) for _ in "qk")
        if c["op"] == "rotate-grad":
            s["dq"], s["dk"] = (_tensor(c, c["tokens"], g, scale=1e-2 if c["dtype"] == "bf16" else 1.0)
                                for _ in "qk")
        return s
    s["q"], s["k"], s["v"], s["do"] = _attention_inputs(c, g)
    if c["op"] != "dense-grad":
        s["blocks"] = _blocks(c, g)
        s["counts"], s["entries"] = _lists(s["blocks"])
    if c["op"] == "layer":
        s.update(_norm_state(_layer_norm(c), c["rows"], g))
    else:
        s["out"], s["lse"] = _forward(c, s)
    return s


def _layer_norm(c):
    """The norm of a 'layer' case: RMS per head, every token rotated."""
    return dict(c, norm="rms", across=False, tokens=c["rows"], offset=0, rotated=c["rows"], pairs="interleaved")


# ------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits
# ------------------------------------------------------------------------------------
def _turn(c, s, x, back=False):
    """x (B,H,S,D) fp32 with the tokens [offset, offset + rotated) rotated, or rotated back."""
    if not c["rotated"]:
        return x
    cos, sin = s["cos"], -s["sin"] if back else s["sin"]
    y = x.clone()
    t = slice(c["offset"], c["offset"] + c["rotated"])
    if c["pairs"] == "interleaved":
        a, b = x[:, :, t, 0::2], x[:, :, t, 1::2]
        y[:, :, t, 0::2] = a * cos[:, 0::2] - b * sin[:, 1::2]
        y[:, :, t, 1::2] = b * cos[:, 0::2] + a * sin[:, 1::2]
    else:
        a, b = x[:, :, t].chunk(2, dim=-1)
        y[:, :, t] = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return y


def _normed(c, x):
    """(normalised x, 1 / its size) of fp32 x (B,H,S,D), over D or over all heads' D."""
    over = (1, 3) if c["across"] else (3,)
    if c["norm"] == "layer":
        x = x - x.mean(dim=over, keepdim=True)
    r = 1.0 / (x.square().mean(dim=over, keepdim=True) + 1e-6).sqrt()
    return x * r, r


def _affine(c, w):
    """A weight or bias in a shape that multiplies (B,H,S,D)."""
    return w.float().view(c["heads"], 1, c["dim"]) if c["across"] else w.float()


def _plain_rotate(c, s, x, w, b):
    y = x.float()
    if c["norm"] != "none":
        y = _normed(c, y)[0] * _affine(c, w)
        if b is not None:
            y = y + _affine(c, b)
    return _turn(c, s, y).to(x.dtype)


def _plain_rotate_grad(c, s, x, dy, w, b):
    """(dx, dw, db); the sums over tokens in 64 bits."""
    d = _turn(c, s, dy.float(), back=True)
    if c["norm"] == "none":
        return d.to(x.dtype), None, None
    n, r = _normed(c, x.float())
    over = (0, 2) if c["across"] else (0, 1, 2)
    dw = (d * n).sum(dim=over, dtype=torch.float64).float().flatten()
    db = None if b is None else d.sum(dim=over, dtype=torch.float64).float().flatten()
    d = d * _affine(c, w)
    over = (1, 3) if c["across"] else (3,)
    dx = d - n * (d * n).mean(dim=over, keepdim=True)
    if c["norm"] == "layer":
        dx = dx - d.mean(dim=over, keepdim=True)
    return (dx * r).to(x.dtype), dw, db


def _weights(c, s, q, k, keep):
    p = q.float() @ k.float().transpose(2, 3)
    p.mul_(c["dim"] ** -0.5)
    if keep is not None:
        p.masked_fill_(~keep, float("-inf"))
    top = p.amax(dim=-1, keepdim=True).clamp_min(-1e30)  # finite where a row keeps nothing
    p.sub_(top).exp_()
    return p.div_(p.sum(dim=-1, keepdim=True).clamp_min(1e-30))


def _plain_attention_grads(c, q, k, v, do, p):
    d = do.float()
    dv = p.transpose(2, 3) @ d
    ds = d @ v.float().transpose(2, 3)
    ds.sub_((p * ds).sum(dim=-1, keepdim=True)).mul_(p).mul_(c["dim"] ** -0.5)
    dq = ds @ k.float()
    dk = ds.transpose(2, 3) @ q.float()
    return dq.to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


def _plain(c, s):
    if c["op"] == "rotate":
        return (_plain_rotate(c, s, s["q"], s["wq"], s["bq"]), _plain_rotate(c, s, s["k"], s["wk"], s["bk"]))
    if c["op"] == "rotate-grad":
        return (_plain_rotate_grad(c, s, s["q"], s["dq"], s["wq"], s["bq"])
                + _plain_rotate_grad(c, s, s["k"], s["dk"], s["wk"], s["bk"]))
    if c["op"] == "dense-grad":
        return _plain_attention_grads(c, s["q"], s["k"], s["v"], s["do"],
                                      _weights(c, s, s["q"], s["k"], None))
    keep = _token_mask(c, s["blocks"])
    if c["op"] == "sparse-grad":
        return _plain_attention_grads(c, s["q"], s["k"], s["v"], s["do"],
                                      _weights(c, s, s["q"], s["k"], keep))
    n = _layer_norm(c)
    q, k = _plain_rotate(n, s, s["q"], s["wq"], None), _plain_rotate(n, s, s["k"], s["wk"], None)
    p = _weights(c, s, q, k, keep)
    out = (p @ s["v"].float()).to(q.dtype)
    dq, dk, dv = _plain_attention_grads(c, q, k, s["v"], s["do"], p)
    dq, dwq, _ = _plain_rotate_grad(n, s, s["q"], dq, s["wq"], None)
    dk, dwk, _ = _plain_rotate_grad(n, s, s["k"], dk, s["wk"], None)
    return out, dq, dk, dv, dwq.to(q.dtype), dwk.to(q.dtype)


# ------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------
def _norm_args(c, s):
    return dict(norm=c["norm"], across_heads=c["across"], eps=1e-6, q_weight=s["wq"], k_weight=s["wk"],
                q_bias=s["bq"], k_bias=s["bk"], cos=s["cos"], sin=s["sin"], rope_offset=c["offset"],
                interleaved=c["pairs"] == "interleaved")


def _own(c, s):
    import mod_dit_amd as md
    from mod_dit_amd import ops

    if c["op"] == "rotate":
        return ops.qk_norm_rope(s["q"], s["k"], **_norm_args(c, s))
    if c["op"] == "rotate-grad":
        dq, dk, dwq, dwk, dbq, dbk = ops.qk_norm_rope_bwd(s["q"], s["k"], s["dq"], s["dk"], **_norm_args(c, s))
        return dq, dwq, dbq, dk, dwk, dbk
    if c["op"] == "dense-grad":
        return ops.flash_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["do"])
    tiles = ops.TileList(s["counts"], s["entries"], 64, c["union"], c["origin"])
    if c["op"] == "sparse-grad":
        return ops.block_sparse_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["do"], tiles)
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "wq", "wk")]
    q, k, v, wq, wk = leaves
    q, k = md.qk_norm_rope(q, k, **dict(_norm_args(_layer_norm(c), s), q_weight=wq, k_weight=wk))
    out = md.block_sparse_attention(q, k, v, tiles)
    return (out.detach(), *torch.autograd.grad(out, leaves, s["do"]))


def run(state):
    return _own(state["c"], state) if own else _plain(state["c"], state)


# ------------------------------------------------------------------------------------
# work, exact results
# ------------------------------------------------------------------------------------
def _density(c):
    """Share of the (row, key) pairs that a mask of this case keeps."""
    return 1.0 if c["op"] == "dense-grad" else c["keep"]


def work(case):
    c = case
    if c["op"].startswith("rotate"):
        tensors = {"rotate": 4, "rotate-grad": 6}[c["op"]]
        n = c["batch"] * c["heads"] * c["tokens"] * c["dim"]
        table = 4.0 * c["rotated"] * c["dim"]  # one cos and one sin per pair
        return {"bytes": 2.0 * tensors * n + table, "flops": 8.0 * tensors * n}
    B, H, D = c["batch"], c["heads"], c["dim"]
    pairs = _density(c) * B * H * c["rows"] * c["keys"]
    tokens = 2.0 * B * H * D * (4 * c["rows"] + 4 * c["keys"]) + 4.0 * B * H * c["rows"]
    if c["op"] == "layer":  # the norm's four and six tensors, attention's, its gradients'
        return {"bytes": 2.0 * B * H * D * c["rows"] * (10 + 4 + 8), "flops": 14.0 * D * pairs}
    return {"bytes": tokens, "flops": 10.0 * D * pairs}


def _exact_rotate(c, s, x, w, b):
    """Norm, weight and rotation of fp64 x, by their definitions."""
    B, H, S, D = x.shape
    y = x
    if c["norm"] != "none":
        rows = y.transpose(1, 2).reshape(B, S, H * D) if c["across"] else y
        if c["norm"] == "layer":
            rows = rows - rows.mean(-1, keepdim=True)
        rows = rows / torch.sqrt((rows * rows).mean(-1, keepdim=True) + 1e-6) * w
        if b is not None:
            rows = rows + b
        y = rows.view(B, S, H, D).transpose(1, 2) if c["across"] else rows
    if not c["rotated"]:
        return y
    lo, hi = c["offset"], c["offset"] + c["rotated"]
    cos, sin = s["cos"].double(), s["sin"].double()
    if c["pairs"] == "interleaved":
        z = torch.view_as_complex(y[:, :, lo:hi].reshape(B, H, hi - lo, D // 2, 2).contiguous())
        z = z * torch.complex(cos[:, ::2], sin[:, ::2])
        turned = torch.view_as_real(z).reshape(B, H, hi - lo, D)
    else:
        z = torch.complex(y[:, :, lo:hi, :D // 2].contiguous(), y[:, :, lo:hi, D // 2:].contiguous())
        z = z * torch.complex(cos, sin)
        turned = torch.cat([z.real, z.imag], dim=-1)
    return torch.cat([y[:, :, :lo], turned, y[:, :, hi:]], dim=2)


def _exact_one(c, s, x, w, b, dy):
    x, w, b = (None if t is None else t.double().requires_grad_(dy is not None) for t in (x, w, b))
    y = _exact_rotate(c, s, x, w, b)
    if dy is None:
        return y
    got = iter(torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy.double()))
    return tuple(None if t is None else next(got) for t in (x, w, b))


def _exact_attention(c, q, k, v, keep):
    x = (q @ k.T) / math.sqrt(c["dim"])
    if keep is not None:
        x = torch.where(keep, x, -torch.inf)
        x = torch.where(keep.any(-1, keepdim=True), x, 0.0)
    p = torch.softmax(x, dim=-1)
    if keep is not None:
        p = p * keep.any(-1, keepdim=True)
    return p @ v


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "rotate":
        return (_exact_one(c, s, s["q"], s["wq"], s["bq"], None), _exact_one(c, s, s["k"], s["wk"], s["bk"], None))
    if c["op"] == "rotate-grad":
        return (_exact_one(c, s, s["q"], s["wq"], s["bq"], s["dq"])
                + _exact_one(c, s, s["k"], s["wk"], s["bk"], s["dk"]))
    n = _layer_norm(c)
    outs = [torch.empty(s[name].shape, device="cuda", dtype=torch.float64) for name in ("q", "q", "k", "v")]
    dw = [torch.zeros(c["dim"], device="cuda", dtype=torch.float64) for _ in "qk"]
    for b in range(c["batch"]):
        for h in range(c["heads"]):
            q, k, v = leaves = [s[name][b, h].double().requires_grad_() for name in ("q", "k", "v")]
            if c["op"] == "layer":
                leaves += [s[name].double().requires_grad_() for name in ("wq", "wk")]
                q = _exact_rotate(n, s, q[None, None], leaves[3], None)[0, 0]
                k = _exact_rotate(n, s, k[None, None], leaves[4], None)[0, 0]
            keep = _token_mask(c, s["blocks"], slice(h, h + 1))[0] if "blocks" in s else None
            out = _exact_attention(c, q, k, v, keep)
            got = torch.autograd.grad(out, leaves, s["do"][b, h].double())
            for to, t in zip(outs, (out.detach(), *got[:3])):
                to[b, h] = t
            for to, t in zip(dw, got[3:]):
                to += t
    return (*outs, *dw) if c["op"] == "layer" else tuple(outs[1:])
