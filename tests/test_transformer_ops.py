"""Attention with a learned relative position bias, cross attention and gated residual norms against plain forms in 64 bits.

The tolerances count roundings: a bf16 rounding is off by at most 2^-8 of its value.  The attention kernels round P (for P V and
P^T dO), dS (for dS K and dS^T Q) and each output once, and D = dO . O carries the error of the rounded O; every bound below is
that sum of absolute values, element by element, plus 2^-13 of the same absolute sums for what is done in 32 bits (products of
up to 128 terms, scores up to 2^6 whose error an exponential passes on as a relative one: 2^6 * 2^7 * 2^-24 * a margin of 16)."""
import math

import pytest
import torch

import pytorch_distributed_training_amd as pdt
from pytorch_distributed_training_amd.nn import functional as F

U = torch.finfo(torch.bfloat16).eps / 2
SLACK = 2.0 ** -13
TINY = 1e-30
gpu = pytest.mark.gpu


def _dev(device):
    if device == "cuda":
        pdt.require_native()
    return torch.device(device)


def _rand(g, *shape, std=1.0, dtype=torch.bfloat16, device="cpu"):
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(device)


def _within(got, want, bound, what):
    got, want, bound = got.double().cpu(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert (over <= TINY).all(), f"{what}: {int((over > TINY).sum())} of {got.numel()} off, worst by {over.max():.3e}"


# ----------------------------------------------------------------------------------------- the plain form in 64 bits
def _attention64(q, k, v, bias, key_live, row_live, do):
    """q [B,H,Sq,hd] ... in 64 bits; masks [B,Sk] / [B,Sq] -> out, dq, dk, dv, dS and the bounds of the first four"""
    scale = q.shape[-1] ** -0.5
    s = q @ k.transpose(-1, -2) * scale
    if bias is not None:
        s = s + bias
    s = s.masked_fill(~key_live[:, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(*s.shape[:-1], 1)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300) * row_live[:, None, :, None]
    out = p @ v
    spread = p @ v.abs()
    e_out = U * (out.abs() + spread) + SLACK * spread
    dp = do @ v.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    e_d = (do.abs() * e_out).sum(-1, keepdim=True)
    e_ds = U * ds.abs() + p * (e_d + SLACK * (do.abs() @ v.abs().transpose(-1, -2)))
    dq, dk, dv = ds @ k * scale, ds.transpose(-1, -2) @ q * scale, p.transpose(-1, -2) @ do
    e_dq = U * dq.abs() + scale * (e_ds @ k.abs())
    e_dk = U * dk.abs() + scale * (e_ds.transpose(-1, -2) @ q.abs())
    e_dv = U * dv.abs() + (U + SLACK) * (p.transpose(-1, -2) @ do.abs())
    return (out, dq, dk, dv, ds, p), (e_out, e_dq, e_dk, e_dv)


def _live(lengths, b, n, device):
    if lengths is None:
        return torch.ones(b, n, dtype=torch.bool, device=device)
    return torch.arange(n, device=device) < torch.tensor(lengths, device=device)[:, None]


def _rel_case(device, b, codes, heads, hd, lengths=None, seed=0, table=None, poison=False):
    g = torch.Generator().manual_seed(seed)
    qc, kc, of = (t.to(device) for t in codes)
    n = qc.numel()
    qkv = _rand(g, b, n, 3 * heads * hd, device=device)
    if table is None:
        table = _rand(g, int(of.max()) + 1, heads, dtype=torch.float32)
    table = table.to(device)
    do = _rand(g, b, n, heads * hd, std=0.1, device=device)
    live = _live(lengths, b, n, device)
    clean = qkv.double() * live[..., None], do.double() * live[..., None]
    if poison:  # what stands behind the last token is not to be read
        qkv = qkv.masked_fill(~live[..., None], math.nan)
        do = do.masked_fill(~live[..., None], math.inf)
    return qkv, table, qc, kc, of, do, live, clean


def _check_rel(device, b, codes, heads, hd, lengths=None, seed=0, table=None, poison=False):
    qkv, table, qc, kc, of, do, live, (qkv64, do64) = _rel_case(device, b, codes, heads, hd, lengths, seed, table, poison)
    n = qc.numel()
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    leaf, tleaf = qkv.clone().requires_grad_(), table.clone().requires_grad_()
    out = F.rel_bias_attention(leaf, tleaf, qc, kc, of, heads, lens)
    dqkv, dtable = torch.autograd.grad(out, [leaf, tleaf], do)
    with torch.no_grad():
        only = F.rel_bias_attention(qkv, table, qc, kc, of, heads, lens)
    q, k, v = qkv64.view(b, n, 3, heads, hd).permute(2, 0, 3, 1, 4)
    bucket = of.long()[(qc.long()[:, None] - kc.long()[None]).clamp(0, of.numel() - 1)]
    real = (bucket >= 0) & (bucket < table.shape[0])
    bias = torch.where(real, table.double()[bucket.clamp(0, table.shape[0] - 1)].permute(2, 0, 1), 0.0)
    do4 = do64.view(b, n, heads, hd).transpose(1, 2)
    (o, dq, dk, dv, ds, p), es = _attention64(q, k, v, bias, live, live.double(), do4)

    def flat(t):
        return t.transpose(1, 2).reshape(b, n, heads * hd)

    _within(out, flat(o), flat(es[0]), "out")
    _within(only, flat(o), flat(es[0]), "out without gradients")
    for i, (name, w, e) in enumerate((("dq", dq, es[1]), ("dk", dk, es[2]), ("dv", dv, es[3]))):
        _within(dqkv[..., i * heads * hd:(i + 1) * heads * hd], flat(w), flat(e), name)
    # the table's gradient is kept in 32 bits: P and O come in two halves (2^-16 each), the sums have up to n * b terms
    err = p * (2.0 ** -15 * (do4.abs() * (o.abs() + p @ v.abs())).sum(-1, keepdim=True) + SLACK / 8 * (do4.abs() @ v.abs().transpose(-1, -2)))

    def by_bucket(t):
        z = torch.zeros(table.shape[0], heads, dtype=torch.float64, device=t.device)
        return z.index_add_(0, bucket.clamp(0, table.shape[0] - 1).reshape(-1), (t.sum(0) * real).reshape(heads, -1).t().contiguous())

    _within(dtable, by_bucket(ds), by_bucket(err) + 2.0 ** -20 * by_bucket(ds.abs()), "dtable")
    return out, dqkv, dtable


def _check_cross(device, b, nq, nk, heads, kv_heads, hd, lengths=None, seed=0, poison=False, grads=True):
    g = torch.Generator().manual_seed(seed)
    q = _rand(g, b, nq, heads * hd, device=device)
    kv = _rand(g, b, nk, 2 * kv_heads * hd, device=device)
    do = _rand(g, b, nq, heads * hd, std=0.1, device=device)
    live = _live(lengths, b, nk, device)
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device)
    kv64 = kv.double() * live[..., None]
    if poison:
        kv = kv.masked_fill(~live[..., None], math.nan)
    q4 = q.double().view(b, nq, heads, hd).transpose(1, 2)
    k1, v1 = kv64.view(b, nk, 2, kv_heads, hd).permute(2, 0, 3, 1, 4)
    k4, v4 = (t.repeat_interleave(heads // kv_heads, 1) for t in (k1, v1))
    rows = torch.ones(b, nq, dtype=torch.float64, device=device)
    (o, dq, dk, dv, _, _), es = _attention64(q4, k4, v4, None, live, rows, do.double().view(b, nq, heads, hd).transpose(1, 2))

    def flat(t):
        return t.transpose(1, 2).reshape(b, nq, heads * hd)

    def shared(t):  # the query heads of a key head add up
        return t.view(b, kv_heads, -1, nk, hd).sum(2).transpose(1, 2).reshape(b, nk, kv_heads * hd)

    with torch.no_grad():
        _within(F.cross_attention(q, kv, heads, kv_heads, lens), flat(o), flat(es[0]), "out without gradients")
    if not grads:
        return
    ql, kl = q.clone().requires_grad_(), kv.clone().requires_grad_()
    out = F.cross_attention(ql, kl, heads, kv_heads, lens)
    gq, gkv = torch.autograd.grad(out, [ql, kl], do)
    _within(out, flat(o), flat(es[0]), "out")
    _within(gq, flat(dq), flat(es[1]), "dq")
    w = kv_heads * hd
    _within(gkv[..., :w], shared(dk), shared(es[2]), "dk")
    _within(gkv[..., w:], shared(dv), shared(es[3]), "dv")
    return out, gq, gkv


def _check_norm(device, shape, per_sample, post, scale, seed=0, only=None):
    g = torch.Generator().manual_seed(seed)
    d = shape[-1]
    x, y = _rand(g, *shape, std=2.0, device=device), _rand(g, *shape, device=device)
    du, dn = _rand(g, *shape, std=0.1, device=device), _rand(g, *shape, std=0.1, device=device)
    gate = _rand(g, *((shape[0], d) if per_sample else (d,)), std=0.5, dtype=torch.float32, device=device)
    ps = [1 + _rand(g, d, std=0.2, dtype=torch.float32, device=device) if i % 2 == 0 else _rand(g, d, dtype=torch.float32, device=device)
          for i in range(4 if post else 2)]
    leaves = [t.clone().requires_grad_() for t in (x, y, gate, *ps)]
    new, normed = F.gated_residual_norm(*leaves[:5], 1e-6, *(leaves[5:] if post else ()), residual_scale=scale)
    with torch.no_grad():
        again = F.gated_residual_norm(x, y, gate, *ps[:2], 1e-6, *(ps[2:] if post else ()), residual_scale=scale)
    assert torch.equal(again[0], new) and torch.equal(again[1], normed)
    w64 = [t.detach().double().requires_grad_() for t in leaves]
    X, Y, G, W, Bi = w64[:5]
    z = torch.nn.functional.layer_norm(Y, (d,), w64[5], w64[6], 1e-6) if post else Y
    Gb = G.view(shape[0], *[1] * (len(shape) - 2), d) if per_sample else G
    u = scale * X + Gb * z
    n = torch.nn.functional.layer_norm(u, (d,), W, Bi, 1e-6)
    outs, gs = (new, normed), (du, dn)
    if only is not None:
        outs, gs, u_n, g64 = (outs[only],), (gs[only],), ((u, n)[only],), (gs[only].double(),)
    else:
        u_n, g64 = (u, n), (du.double(), dn.double())
    got = torch.autograd.grad(outs, leaves, gs, allow_unused=True)
    want = torch.autograd.grad(u_n, w64, g64, allow_unused=True)
    # one rounding of each bf16 output; 32-bit work on rows of d terms is off by some 2^-24 * sqrt(d) of the row's largest
    # value, times 1 / deviation where a norm divides by it: 2^-17 of the row's largest output covers widths up to 2048
    for name, a, b in (("x_new", new, u), ("normed", normed, n)):
        b = b.detach()
        _within(a, b, U * b.abs() + 2.0 ** -17 * b.abs().amax(-1, keepdim=True), name)
    names = ("dx", "dbranch", "dgate", "dweight", "dbias", "dpost_weight", "dpost_bias")
    rows = math.prod(shape[:-1])
    for i, (name, a, b) in enumerate(zip(names, got, want)):
        if b is None or a is None:
            assert b is None or not b.abs().max() > 0, name
            assert a is None or not a.abs().max() > 0, name
            continue
        if i < 2:
            _within(a, b, U * b.abs() + 2.0 ** -16 * b.abs().amax(-1, keepdim=True), name)
        else:  # sums over the rows in 32 bits of terms whose own error is 2^-17 of the largest
            _within(a, b, 2.0 ** -17 * b.abs().max() + 2.0 ** -17 * math.sqrt(rows) * 0.2 + TINY, name)


def _grid(side):
    return pdt.nn.grid_position_buckets(side, side, prefix=1)


def _log(n, far=16, buckets=8):
    return pdt.nn.log_position_buckets(n, buckets, far)


# ------------------------------------------------------------------------------------------------- on the CPU
def test_grid_position_buckets():
    q, k, of = pdt.nn.grid_position_buckets(3, 2, prefix=1)
    assert of.tolist() == list(range(5 * 3 + 3))
    b = of[(q[:, None] - k[None]).clamp(0, of.numel() - 1).long()]
    yx = [(i // 2, i % 2) for i in range(6)]
    seen = {}
    for i, (yi, xi) in enumerate(yx):
        for j, (yj, xj) in enumerate(yx):
            seen.setdefault(int(b[i + 1, j + 1]), set()).add((yi - yj, xi - xj))
    assert len(seen) == 15 and all(len(v) == 1 for v in seen.values())
    prefix = {int(b[0, 0])}, set(b[0, 1:].tolist()), set(b[1:, 0].tolist())
    assert all(len(s) == 1 for s in prefix) and len(set.union(*prefix, set(seen))) == 18


def test_log_position_buckets():
    q, k, of = pdt.nn.log_position_buckets(300, 32, 128)
    b = of[(q[:, None] - k[None]).clamp(0, of.numel() - 1).long()]
    assert b[10, 10] == 0 and b[10, 3] == 7 and b[10, 11] == 17 and b[299, 0] == 15 and b[0, 299] == 31
    assert b.min() == 0 and b.max() == 31 and (torch.diff(b[299].flip(0)[:200]) >= 0).all()
    q, k, of = pdt.nn.log_position_buckets(40, 32, 128, bidirectional=False)
    b = of[(q[:, None] - k[None]).clamp(0, of.numel() - 1).long()]
    assert (b.triu() == 0).all() and b[20, 5] == 15 and b[39, 0] > 16


CPU_REL = [dict(b=2, codes=_grid(3), heads=2, hd=8), dict(b=4, codes=_log(17), heads=3, hd=4, lengths=[17, 9, 1, 0], poison=True)]


@pytest.mark.parametrize("case", CPU_REL)
def test_rel_bias_attention_oracle(case):
    _check_rel(_dev("cpu"), **case)


@pytest.mark.parametrize("case", [dict(b=2, nq=5, nk=7, heads=4, kv_heads=2, hd=8),
                                  dict(b=3, nq=1, nk=9, heads=3, kv_heads=1, hd=4, lengths=[9, 4, 0], poison=True)])
def test_cross_attention_oracle(case):
    _check_cross(_dev("cpu"), **case)


@pytest.mark.parametrize("per_sample,post", [(False, True), (True, False), (True, True)])
def test_gated_residual_norm_oracle(per_sample, post):
    _check_norm(_dev("cpu"), (3, 5, 20), per_sample, post, 0.5)


def test_gradients_against_differences():
    """Central differences in 64 bits through the oracle's formulas."""
    g = torch.Generator().manual_seed(3)

    def r(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()

    qc, kc, of = _grid(2)
    lens = torch.tensor([5, 3])
    assert torch.autograd.gradcheck(lambda a, t: F.rel_bias_attention(a, t, qc, kc, of, 2, lens), (r(2, 5, 24), r(int(of.max()) + 1, 2)))
    assert torch.autograd.gradcheck(lambda a, b: F.cross_attention(a, b, 4, 2, lens), (r(2, 3, 16), r(2, 6, 16)))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_refusals(device):
    dev = _dev(device)
    qc, kc, of = (t.to(dev) for t in _grid(2))
    qkv, table = torch.zeros(2, 5, 96, dtype=torch.bfloat16, device=dev), torch.zeros(12, 1, device=dev)

    def rel(qkv=qkv, table=table, qc=qc, kc=kc, of=of, heads=1, lens=None):
        return F.rel_bias_attention(qkv, table, qc, kc, of, heads, lens)

    assert rel().shape == (2, 5, 32)
    lens = torch.tensor([5, 2], device=dev)
    assert rel(lens=lens).shape == (2, 5, 32)
    for bad in (dict(qkv=qkv[0]), dict(heads=5), dict(heads=0), dict(table=table[:, 0]), dict(table=table.expand(12, 3)), dict(qc=qc[:4]),
                dict(kc=kc[None]), dict(of=of[:0]), dict(qc=qc.float()), dict(lens=lens[:1]), dict(lens=lens.float())):
        with pytest.raises(ValueError):
            rel(**bad)
    q, kv = torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=dev), torch.zeros(2, 7, 64, dtype=torch.bfloat16, device=dev)
    assert F.cross_attention(q, kv, 2, 1).shape == q.shape
    for bad in ((q, kv, 2, 3), (q, kv, 0, 1), (q, kv, 2, 2), (q[:1], kv, 2, 1), (q[0], kv[0], 2, 1), (q.float(), kv, 2, 1),
                (q, kv, 2, 1, lens[:1]), (q, kv, 3, 1)):
        with pytest.raises(ValueError):
            F.cross_attention(*bad)
    x, v = torch.zeros(2, 3, 8, dtype=torch.bfloat16, device=dev), torch.ones(8, device=dev)
    assert F.gated_residual_norm(x, x, v, v, v)[0].shape == x.shape
    for bad in ((x, x[:1], v, v, v), (x, x.float(), v, v, v), (x, x, v[:4], v, v), (x, x, v.expand(3, 8), v, v), (x, x, v, v[:4], v),
                (x, x, v, v, v, 1e-6, v), (x, x, v, v, v, 1e-6, v, v[:1])):
        with pytest.raises(ValueError):
            F.gated_residual_norm(*bad)
    if device == "cuda":
        for bad in (dict(lens=lens.cpu()), dict(table=table.cpu()), dict(of=of.cpu())):
            with pytest.raises(ValueError):
                rel(**bad)


OPTIONS = dict(rel_pos_bias=True, layer_scale=0.5, post_norm=True, pool="attention")


def test_vit_options_leave_the_plain_model_alone():
    from pytorch_distributed_training_amd.models import build_model

    plain, more = build_model("vit_tiny_test"), build_model("vit_tiny_test", **OPTIONS)
    assert set(plain.state_dict()) < set(more.state_dict())
    new = sorted(set(more.state_dict()) - set(plain.state_dict()))
    assert "encoder.layers.encoder_layer_0.self_attention.relative_position_bias_table" in new and "pool.query" in new
    assert not any("codes" in k or "bucket" in k for k in more.state_dict())
    for bad in (dict(pool="mean"), dict(post_norm=True)):
        with pytest.raises(ValueError):
            build_model("vit_tiny_test", **bad)


def _vit_gradients(model, x, y):
    loss = torch.nn.functional.cross_entropy(model(x).float(), y)
    return loss.detach(), torch.autograd.grad(loss, list(model.parameters()))


@pytest.mark.parametrize("options", [OPTIONS, dict(rel_pos_bias=True), dict(layer_scale=0.1), dict(pool="attention"), dict(OPTIONS, dropout=0.2)], ids=str)
def test_vit_with_options_has_every_gradient(options):
    from pytorch_distributed_training_amd.models import build_model

    torch.manual_seed(0)
    m = build_model("vit_tiny_test", num_classes=10, **options)
    for p in m.parameters():  # (the head and the tables start at zero)
        torch.nn.init.normal_(p, std=0.1)
    loss, gs = _vit_gradients(m, torch.rand(3, 3, 32, 32), torch.tensor([1, 2, 3]))
    assert torch.isfinite(loss)
    for (name, _), g in zip(m.named_parameters(), gs):
        assert torch.isfinite(g).all() and g.abs().max() > 0, name


@gpu
def test_vit_with_options_against_the_oracle():
    """Logits and every gradient of a model with all options, kernels against the fp32 formulas on the same bf16 activations."""
    from pytorch_distributed_training_amd import ops
    from pytorch_distributed_training_amd.models import build_model

    dev = _dev("cuda")
    torch.manual_seed(0)
    m = build_model("vit_ti_16", num_classes=16, image_size=112, **OPTIONS).to(dev)
    for n, p in m.named_parameters():
        if n.endswith("bias_table") or n.startswith("heads"):
            torch.nn.init.normal_(p, std=0.1)
    g = torch.Generator().manual_seed(1)
    x = torch.rand(4, 3, 112, 112, generator=g).to(dev).to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    y = torch.randint(0, 16, (4,), generator=g).to(dev)
    before = dict(F.fallback_counts)
    loss, gs = _vit_gradients(m, x, y)
    assert dict(F.fallback_counts) == before
    ops.set_force_reference(True)
    try:
        want, ws = _vit_gradients(m, x, y)
    finally:
        ops.set_force_reference(False)
    assert abs(loss - want) <= 16 * U * abs(want)
    true = _vit_gradients(m, x.float(), y)[1]  # the same formulas in 32 bits throughout
    for (name, _), a, b, c in zip(m.named_parameters(), gs, ws, true):
        # Twelve layers of some ten roundings each, each off by U at most and by U / sqrt(3) in the mean square, add up to
        # sqrt(120 / 3) U of a gradient's norm where they meet at random.  Where the gradient itself is a small difference
        # (pool.query: the sum over the keys of P (dP - D) k, whose P (dP - D) add up to zero) the same roundings are
        # (sum P |dP| |k|) / |sum P (dP - D) k| times as large against its norm, for the kernels and the oracle alike.  So the
        # kernels are held to the oracle's own error: they round P and dS too, 12 roundings a layer for 10, which is
        # sqrt(1.2) = 1.1 times its error, and two independent errors' norms of this many terms differ by less than that again.
        size, off, oracle = c.double().norm(), (a.double() - c.double()).norm(), (b.double() - c.double()).norm()
        assert off <= 2 * max(oracle, math.sqrt(40) * U * size / 2) + 1e-12, (name, off, oracle, size)


@gpu
def test_engine_trains_a_vit_with_options():
    from pytorch_distributed_training_amd import dist as pdist
    from pytorch_distributed_training_amd.engine import Engine, EngineConfig

    import os

    _dev("cuda")
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29541")
    pdist.init_process_group(backend="rccl", local_rank=0)
    eng = Engine(EngineConfig(model="vit_tiny_test", num_classes=10, optimizer="adamw", lr=1e-3, sync_bn=False, seed=0,
                              model_options=OPTIONS))
    g = torch.Generator().manual_seed(0)
    x, y = torch.rand(8, 3, 32, 32, generator=g).cuda(), torch.randint(0, 10, (8,), generator=g).cuda()
    before = dict(F.fallback_counts)
    start = [p.detach().clone() for p in eng.net.parameters()]
    losses = [float(eng.train_step(x, y)) for _ in range(3)]
    assert all(math.isfinite(v) for v in losses)
    assert all(not torch.equal(a, b) for a, b in zip(start, eng.net.parameters()))
    assert dict(F.fallback_counts) == before


# ------------------------------------------------------------------------------------------------- on the GPU
REL = [
    dict(b=1, codes=_log(1), heads=1, hd=64), dict(b=2, codes=_log(2), heads=2, hd=32), dict(b=3, codes=_grid(2), heads=3, hd=128),
    dict(b=2, codes=_log(31), heads=2, hd=64), dict(b=2, codes=_log(32), heads=1, hd=32), dict(b=2, codes=_log(33), heads=1, hd=128),
    dict(b=2, codes=_log(63), heads=3, hd=64), dict(b=1, codes=_log(64), heads=2, hd=64), dict(b=2, codes=_log(65), heads=2, hd=128),
    dict(b=2, codes=_log(129, 200, 32), heads=2, hd=64), dict(b=3, codes=_grid(14), heads=3, hd=64), dict(b=2, codes=_grid(15), heads=2, hd=64),
    dict(b=300, codes=_grid(4), heads=2, hd=64), dict(b=2, codes=_grid(24), heads=2, hd=64), dict(b=1, codes=_grid(17), heads=2, hd=32),
    dict(b=5, codes=_grid(14), heads=2, hd=64, lengths=[197, 0, 1, 64, 130], poison=True),
    dict(b=4, codes=_log(300, 64, 32), heads=2, hd=128, lengths=[300, 2, 0, 257], poison=True),
    dict(b=4, codes=_log(100, 20, 8), heads=3, hd=32, lengths=[33, 100, 96, 1], poison=True),
    dict(b=1, codes=_log(2049, 128, 32), heads=1, hd=64), dict(b=2, codes=_log(1100, 2000, 32), heads=1, hd=128, lengths=[1100, 700]),
]


@gpu
@pytest.mark.parametrize("case", REL, ids=lambda c: f"b{c['b']}-n{c['codes'][0].numel()}-h{c['heads']}x{c['hd']}{'-ragged' if 'lengths' in c else ''}")
def test_rel_bias_attention(case):
    before = dict(F.fallback_counts)
    _check_rel(_dev("cuda"), **case)
    assert dict(F.fallback_counts) == before


@gpu
def test_rel_bias_forbidden_lowest_and_unnamed_entries():
    """-inf entries forbid pairs (a row may lose every key), the lowest finite value beats nothing but itself, and an entry
    that names no bucket adds nothing and gets no gradient."""
    dev = _dev("cuda")
    n, heads, hd = 70, 2, 64
    qc, kc = torch.arange(n) + n, torch.arange(n)
    of = torch.zeros(2 * n + 1, dtype=torch.int64)
    of[:n] = 1                      # keys after the query
    of[n + 5] = 2
    of[n + 9], of[n + 11] = -1, 77  # no such buckets
    table = torch.tensor([[0.3, -0.2], [-math.inf, 1.0], [torch.finfo(torch.float32).min, 0.5]])
    out, dqkv, dtable = _check_rel_inf(dev, (qc, kc, of), heads, hd, table)
    assert dtable[1, 0] == 0
    # every key forbidden: zeros, and no gradients
    gone = torch.full((1, heads), -math.inf)
    g = torch.Generator().manual_seed(5)
    qkv = _rand(g, 1, n, 3 * heads * hd, device=dev).requires_grad_()
    t = gone.to(dev).requires_grad_()
    zero = torch.zeros_like(of).to(dev)
    o = F.rel_bias_attention(qkv, t, qc.to(dev), kc.to(dev), zero, heads)
    gs = torch.autograd.grad(o, [qkv, t], torch.ones_like(o))
    assert not o.any() and not gs[0].any() and not gs[1].any()
    # every key at the lowest value: as without a bias
    low = torch.full((1, heads), torch.finfo(torch.float32).min).to(dev)
    none = torch.zeros((1, heads)).to(dev)
    with torch.no_grad():
        a = F.rel_bias_attention(qkv, low, qc.to(dev), kc.to(dev), zero, heads)
    v = qkv.detach()[..., 2 * heads * hd:].double().mean(1, keepdim=True)
    assert (a.double() - v).abs().max() < 2 * U * qkv.detach().abs().max()  # equal weights: absorbed scores
    assert torch.isfinite(F.rel_bias_attention(qkv, none, qc.to(dev), kc.to(dev), zero, heads)).all()


def _check_rel_inf(dev, codes, heads, hd, table):
    """`_check_rel` with -inf and lowest entries in the table: the 64-bit form takes them as they are (head 0, buckets 1 and 2)."""
    return _check_rel(dev, 2, codes, heads, hd, table=table)


CROSS = [
    dict(b=1, nq=1, nk=1, heads=1, kv_heads=1, hd=64), dict(b=2, nq=1, nk=33, heads=4, kv_heads=2, hd=32),
    dict(b=2, nq=3, nk=64, heads=8, kv_heads=1, hd=128), dict(b=3, nq=7, nk=31, heads=2, kv_heads=2, hd=64),
    dict(b=2, nq=33, nk=100, heads=2, kv_heads=1, hd=64), dict(b=2, nq=130, nk=65, heads=6, kv_heads=2, hd=32),
    dict(b=1, nq=64, nk=1000, heads=2, kv_heads=1, hd=128), dict(b=1, nq=1, nk=3000, heads=2, kv_heads=2, hd=64),
    dict(b=1, nq=1, nk=5001, heads=8, kv_heads=2, hd=128), dict(b=1, nq=600, nk=40, heads=3, kv_heads=1, hd=64),
    dict(b=4, nq=5, nk=500, heads=3, kv_heads=1, hd=64, lengths=[500, 0, 1, 77], poison=True),
    dict(b=3, nq=50, nk=300, heads=4, kv_heads=4, hd=32, lengths=[64, 300, 0], poison=True),
    dict(b=2, nq=1, nk=4000, heads=4, kv_heads=1, hd=128, lengths=[17, 4000], poison=True),
    dict(b=70, nq=1, nk=197, heads=12, kv_heads=12, hd=64), dict(b=2, nq=11, nk=45, heads=9, kv_heads=3, hd=32, lengths=[45, 1]),
]


@gpu
@pytest.mark.parametrize("case", CROSS, ids=lambda c: f"b{c['b']}-{c['nq']}x{c['nk']}-h{c['heads']}of{c['kv_heads']}x{c['hd']}{'-ragged' if 'lengths' in c else ''}")
def test_cross_attention(case):
    before = dict(F.fallback_counts)
    _check_cross(_dev("cuda"), **case)
    assert dict(F.fallback_counts) == before


NORM = [((1, 1, 4), False, True, 1.0), ((3, 5, 36), True, True, 0.5), ((2, 197, 192), False, True, 1.0), ((7, 768), True, False, 1.0),
        ((4, 33, 1024), True, False, 0.5), ((5, 3, 11, 260), True, True, 0.9), ((2, 9, 2048), False, True, 1.0), ((2, 65, 1300), True, True, 1.0),
        ((1, 2100, 64), True, False, 1.0), ((1300, 2, 40), True, True, 1.0), ((3, 700, 516), False, False, 1.0)]


@gpu
@pytest.mark.parametrize("case", NORM, ids=str)
def test_gated_residual_norm(case):
    before = dict(F.fallback_counts)
    _check_norm(_dev("cuda"), *case)
    assert dict(F.fallback_counts) == before


@gpu
@pytest.mark.parametrize("only", [0, 1])
def test_gated_residual_norm_with_one_gradient(only):
    _check_norm(_dev("cuda"), (2, 37, 128), True, True, 1.0, only=only)


@gpu
def test_empty_inputs():
    dev = _dev("cuda")
    qc, kc, of = (t.to(dev) for t in _log(5))
    t = torch.ones(8, 2, device=dev, requires_grad=True)
    e = torch.zeros(0, 5, 192, dtype=torch.bfloat16, device=dev, requires_grad=True)
    o = F.rel_bias_attention(e, t, qc, kc, of, 2)
    g = torch.autograd.grad(o, [e, t], torch.zeros_like(o))
    assert o.shape == (0, 5, 64) and g[0].shape == e.shape and not g[1].any()
    e = torch.zeros(2, 0, 192, dtype=torch.bfloat16, device=dev)
    assert F.rel_bias_attention(e, t.detach(), qc[:0], kc[:0], of, 2).shape == (2, 0, 64)
    q = torch.ones(2, 3, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    kv = torch.zeros(2, 0, 128, dtype=torch.bfloat16, device=dev, requires_grad=True)
    o = F.cross_attention(q, kv, 2)
    gq, gkv = torch.autograd.grad(o, [q, kv], torch.ones_like(o))
    assert not o.any() and not gq.any() and gkv.shape == kv.shape
    kv = torch.ones(2, 9, 128, dtype=torch.bfloat16, device=dev, requires_grad=True)
    o = F.cross_attention(q[:, :0], kv, 2)
    assert o.shape == (2, 0, 64) and not torch.autograd.grad(o, kv, torch.ones_like(o))[0].any()
    x = torch.zeros(0, 3, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    v = torch.ones(64, device=dev, requires_grad=True)
    a, b = F.gated_residual_norm(x, x, v, v, v)
    assert a.shape == x.shape and not torch.autograd.grad(b, v, torch.zeros_like(b))[0].any()


@gpu
def test_views_other_types_and_alignment():
    """Rows inside a wider tensor, an expanded batch, misaligned slices, int64 codes and lengths, a bf16 table."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(1)
    wide = _rand(g, 2, 50, 64 + 192 + 64, device=dev)
    qc, kc, of = (t.to(dev) for t in _log(50))
    table = _rand(g, 8, 1, dtype=torch.float32, device=dev)
    view = wide[:, :, 64:256]
    args = (table, qc, kc, of, 1)
    with torch.no_grad():
        want = F.rel_bias_attention(view.contiguous(), *args)
        assert torch.equal(F.rel_bias_attention(view, *args), want)
        assert torch.equal(F.rel_bias_attention(wide[:, :, 63:255], *args), F.rel_bias_attention(wide[:, :, 63:255].contiguous(), *args))
        assert torch.equal(F.rel_bias_attention(view.transpose(0, 1).contiguous().transpose(0, 1), *args), want)
        assert torch.equal(F.rel_bias_attention(view, table, qc.long(), kc.long(), of.long(), 1, torch.tensor([50, 50], device=dev)), want)
        lens = torch.tensor([9, 50, 3], dtype=torch.int32, device=dev)[1:]
        a = F.rel_bias_attention(view, *args, lens)
        assert torch.equal(a, F.rel_bias_attention(view, *args, lens.clone()))
        one = view[:1].expand(2, -1, -1)
        assert torch.equal(F.rel_bias_attention(one, *args)[1], want[0])
        q, kv = wide[:, :7, :128], wide[:, :, 64:320]
        want = F.cross_attention(q.contiguous(), kv.contiguous(), 2)
        assert torch.equal(F.cross_attention(q, kv, 2), want)
        assert torch.equal(F.cross_attention(q[:, ::2], kv[:, ::3], 2), F.cross_attention(q[:, ::2].contiguous(), kv[:, ::3].contiguous(), 2))
        x = wide[:, :, 3:71]
        v = _rand(g, 69, dtype=torch.float32, device=dev)[1:]
        a = F.gated_residual_norm(x, x, v, v, v)
        b = F.gated_residual_norm(x.contiguous(), x.contiguous(), v.clone(), v.clone(), v.clone())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = table.bfloat16().requires_grad_()
    o = F.rel_bias_attention(view, t, qc, kc, of, 1)
    (gt,) = torch.autograd.grad(o, t, torch.ones_like(o))
    assert gt.dtype == torch.bfloat16
    # gradients of views and of broadcast inputs
    base = wide.clone().requires_grad_()
    o = F.rel_bias_attention(base[:, :, 64:256], *args)
    (gb,) = torch.autograd.grad(o, base, torch.ones_like(o).expand_as(o))
    leaf = view.clone().requires_grad_()
    (gl,) = torch.autograd.grad(F.rel_bias_attention(leaf, *args), leaf, torch.ones_like(o))
    assert torch.equal(gb[:, :, 64:256], gl) and not gb[:, :, :64].any() and not gb[:, :, 256:].any()


@gpu
def test_types_without_a_kernel_are_counted():
    dev = _dev("cuda")
    before = sum(F.fallback_counts.values())
    q, kv = torch.randn(2, 3, 64, device=dev), torch.randn(2, 5, 128, device=dev)
    F.cross_attention(q, kv, 1)
    F.cross_attention(q.bfloat16(), kv.bfloat16(), 4)  # head_dim 16
    F.gated_residual_norm(q, q, q[0, 0], q[0, 0], q[0, 0])
    qc, kc, of = (t.to(dev) for t in pdt.nn.grid_position_buckets(33, 33))
    F.rel_bias_attention(torch.zeros(1, qc.numel(), 96, dtype=torch.bfloat16, device=dev), torch.zeros(int(of.max()) + 1, 1, device=dev), qc, kc, of, 1)
    assert sum(F.fallback_counts.values()) == before + 4


@gpu
def test_rel_bias_pairs_past_the_reach_of_the_table():
    """More than 2048 positions in a row (the dQ pass looks at 64 tiles of keys at a time), lengths that end inside tiles."""
    _check_rel(_dev("cuda"), 8, _log(2200, 64, 32), 2, 32, lengths=[2200, 2100, 0, 1, 700, 2177, 64, 2113], poison=True)


def _chain(dev, seed):
    """The operators as a model uses them: self attention with positions, a block end, cross attention, a block end."""
    g = torch.Generator().manual_seed(seed)
    b, n, m, heads, hd = 3, 50, 70, 2, 64
    d = heads * hd
    qc, kc, of = (t.to(dev) for t in _grid(7))
    p = dict(qkv=_rand(g, b, n, 3 * d, device=dev), table=_rand(g, int(of.max()) + 1, heads, dtype=torch.float32, device=dev),
             x=_rand(g, b, n, d, device=dev), kv=_rand(g, b, m, 2 * d, device=dev), g1=_rand(g, d, dtype=torch.float32, device=dev),
             g2=_rand(g, b, d, dtype=torch.float32, device=dev), w=1 + _rand(g, d, std=0.1, dtype=torch.float32, device=dev),
             bias=_rand(g, d, dtype=torch.float32, device=dev))
    lens = torch.tensor([70, 33, 0], dtype=torch.int32, device=dev)

    def step(p):
        y = F.rel_bias_attention(p["qkv"], p["table"], qc, kc, of, heads)
        x, h = F.gated_residual_norm(p["x"], y, p["g1"], p["w"], p["bias"], 1e-6, p["w"], p["bias"])
        y = F.cross_attention(h, p["kv"], heads, None, lens)
        x, h = F.gated_residual_norm(x, y, p["g2"], p["w"], p["bias"])
        return [h, *torch.autograd.grad([x, h], list(p.values()), [torch.ones_like(x), torch.ones_like(h)])]

    return {k: v.requires_grad_() for k, v in p.items()}, step


@gpu
def test_chain_against_the_oracle_and_bit_for_bit():
    dev = _dev("cuda")
    p, step = _chain(dev, 0)
    a, b = step(p), step(p)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    from pytorch_distributed_training_amd import ops
    ops.set_force_reference(True)
    try:
        want = step(p)
    finally:
        ops.set_force_reference(False)
    for x, y in zip(a, want):  # a chain of four operators with a handful of roundings each: 2^-8 * 8 in the 2-norm
        assert (x.double() - y.double()).norm() <= 8 * U * y.double().norm()


@gpu
def test_captured_and_replayed_chain():
    dev = _dev("cuda")
    p, step = _chain(dev, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(p)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(p)
        graphs.append((graph, outs))
    for seed in range(3):
        fresh, _ = _chain(dev, 10 + seed)
        with torch.no_grad():
            for k in p:
                p[k].copy_(fresh[k])
        want = [t.clone() for t in step(p)]
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(x, y) for x, y in zip(outs, want))


@gpu
def test_two_streams_at_once():
    dev = _dev("cuda")
    jobs = [_chain(dev, 20 + i) for i in range(2)]
    want = [[t.clone() for t in step(p)] for p, step in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [None, None]
    for _ in range(5):
        for i, (s, (p, step)) in enumerate(zip(streams, jobs)):
            with torch.cuda.stream(s):
                got[i] = step(p)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


@gpu
def test_keys_past_32_bit_offsets():
    """A cache of more than 2^32 bytes for one sequence: the last keys are read, and nothing behind the length."""
    dev = _dev("cuda")
    heads, hd, n = 8, 128, 1_100_003
    kv = torch.zeros(1, n, 2 * heads * hd, dtype=torch.bfloat16, device=dev)
    assert kv.numel() * 2 > 2 ** 32
    q = torch.ones(1, 1, heads * hd, dtype=torch.bfloat16, device=dev)
    kv[0, n - 2, :heads * hd] = 2.0  # score 2 * 128 / sqrt(128) = 22.6: e^22.6 = 6.6e9 against 1.1e6 others
    kv[0, n - 2, heads * hd:] = 3.0
    kv[0, n - 1] = math.nan
    lens = torch.tensor([n - 1], dtype=torch.int32, device=dev)
    share = 1 / (1 + (n - 2) * math.exp(-2 * 128 / math.sqrt(128)))
    with torch.no_grad():
        out = F.cross_attention(q, kv, heads, None, lens)
        wide = F.cross_attention(q.expand(1, 40, -1), kv, heads, None, lens)  # the kernel for more rows
    for o in (out, wide):
        assert (o.double() - 3 * share).abs().max() <= 3 * (2 * U + SLACK)


@gpu
def test_lengths_and_buckets_outside_their_range():
    """Counts below zero are none and counts past the end all, in 64 bits too; a bucket past 32 bits is no bucket."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(2)
    q, kv = _rand(g, 4, 3, 64, device=dev), _rand(g, 4, 40, 128, device=dev)
    want = torch.tensor([0, 40, 40, 7], dtype=torch.int32, device=dev)
    qc, kc, of = (t.to(dev) for t in _log(40))
    qkv, table = _rand(g, 4, 40, 192, device=dev), _rand(g, 8, 1, dtype=torch.float32, device=dev)
    far = of.long()
    far[5] += 2 ** 32  # an entry of bucket_of[5] in its lower half
    none = of.clone()
    none[5] = -1
    for lens in (torch.tensor([-3, 41, 2 ** 31 - 1, 7], dtype=torch.int32, device=dev),
                 torch.tensor([-(2 ** 33) - 1, 2 ** 32, 2 ** 32 + 3, 7], device=dev)):
        a, b = q.clone().requires_grad_(), q.clone().requires_grad_()
        x, y = F.cross_attention(a, kv, 1, None, lens), F.cross_attention(b, kv, 1, None, want)
        assert torch.equal(x, y)
        assert torch.equal(*(torch.autograd.grad(o, t, torch.ones_like(o))[0] for o, t in ((x, a), (y, b))))
        a, b = table.clone().requires_grad_(), table.clone().requires_grad_()
        x, y = F.rel_bias_attention(qkv, a, qc, kc, far, 1, lens), F.rel_bias_attention(qkv, b, qc, kc, none, 1, want)
        assert torch.equal(x, y)
        assert torch.equal(*(torch.autograd.grad(o, t, torch.ones_like(o))[0] for o, t in ((x, a), (y, b))))


@gpu
def test_more_sequences_than_a_launch_has_workgroups():
    dev = _dev("cuda")
    n = 1 << 24
    q, kv = (torch.zeros(1, 1, w, dtype=torch.bfloat16, device=dev).expand(n, -1, -1) for w in (32, 64))
    with pytest.raises(RuntimeError, match="workgroups"):
        F.cross_attention(q, kv, 1)
    qc, kc, of = (t.to(dev) for t in _log(1))
    table = torch.zeros(8, 1, device=dev)
    with pytest.raises(RuntimeError, match="workgroups"):
        F.rel_bias_attention(torch.zeros(1, 1, 96, dtype=torch.bfloat16, device=dev).expand(n, -1, -1), table, qc, kc, of, 1)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_gradients_twice_and_of_gradients(device):
    """A graph that is kept gives the same gradients again; gradients of gradients are refused."""
    dev = _dev(device)
    g = torch.Generator().manual_seed(7)
    qc, kc, of = (t.to(dev) for t in _log(9))
    qkv, q, kv = (_rand(g, 2, 9, w, device=dev).requires_grad_() for w in (192, 64, 128))
    table, gate = (_rand(g, *s, dtype=torch.float32, device=dev).requires_grad_() for s in ((8, 1), (64,)))
    one = torch.ones(64, device=dev)
    for call, leaves in ((lambda: F.rel_bias_attention(qkv, table, qc, kc, of, 1), [qkv, table]),
                         (lambda: F.cross_attention(q, kv, 1), [q, kv]),
                         (lambda: F.gated_residual_norm(q, q * 0.5, gate, one, one)[1], [q, gate])):
        out = call()
        w = torch.ones_like(out)
        w[:, ::2] = 0.5
        a = torch.autograd.grad(out, leaves, w, retain_graph=True)
        b = torch.autograd.grad(out, leaves, w, retain_graph=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        with pytest.raises(RuntimeError):
            c = torch.autograd.grad(out, leaves, w, create_graph=True)
            torch.autograd.grad(c[0].float().sum(), leaves)


@gpu
def test_capture_beside_an_eager_graph_of_the_same_leaves_is_refused():
    """The forward says so: the backward would end the process.  Released, the capture works."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(8)
    qc, kc, of = (t.to(dev) for t in _log(9))
    table, q, gate = (_rand(g, *s, dtype=t, device=dev).requires_grad_()
                      for s, t in (((8, 1), torch.float32), ((2, 9, 64), torch.bfloat16), ((64,), torch.float32)))
    qkv, kv, x = (_rand(g, 2, 9, w, device=dev) for w in (192, 128, 64))
    one = torch.ones(64, device=dev)
    for call, leaf in ((lambda: F.rel_bias_attention(qkv, table, qc, kc, of, 1), table), (lambda: F.cross_attention(q, kv, 1), q),
                       (lambda: F.gated_residual_norm(x, x, gate, one, one)[0], gate)):
        alive = call()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                one * 2
                call()
        want = torch.autograd.grad(alive, leaf, torch.ones_like(alive))[0]
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
            (got,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


ANY_CODES = [dict(n=150, entries=1, buckets=1, hd=64), dict(n=70, entries=2, buckets=3, hd=32), dict(n=150, entries=7, buckets=130, hd=64),
             dict(n=300, entries=4096, buckets=500, hd=128), dict(n=33, entries=4095, buckets=1, hd=64), dict(n=40, entries=5, buckets=0, hd=32)]


@gpu
@pytest.mark.parametrize("case", ANY_CODES, ids=lambda c: f"n{c['n']}-r{c['entries']}-b{c['buckets']}x{c['hd']}")
def test_rel_bias_any_codes(case):
    """Codes and buckets in no order, on both sides of the table's reach, buckets that no entry names and entries without one."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(11)
    n, r, nb = case["n"], case["entries"], case["buckets"]
    qc, kc = (torch.randint(-r, 2 * r + 1, (n,), generator=g) for _ in range(2))
    of = torch.randint(-1, nb + 2, (r,), generator=g)
    table = torch.randn(nb, 3, generator=g)
    if nb == 0:
        qkv = _rand(g, 2, n, 9 * case["hd"], device=dev)
        t = table.to(dev).requires_grad_()
        out = F.rel_bias_attention(qkv, t, qc.to(dev), kc.to(dev), of.to(dev), 3)
        (dt,) = torch.autograd.grad(out, t, torch.ones_like(out))
        assert dt.shape == (0, 3)
        return
    _check_rel(dev, 3, (qc, kc, of), 3, case["hd"], lengths=[n, n // 2, 1], table=table, poison=True)


@gpu
def test_gradients_of_one_input_alone():
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(12)
    qc, kc, of = (t.to(dev) for t in _grid(6))
    qkv = _rand(g, 3, 37, 384, device=dev)
    table = _rand(g, 2, int(of.max()) + 1, dtype=torch.float32, device=dev).t()  # (columns that are not neighbours)
    w = _rand(g, 3, 37, 128, device=dev)
    a, t = qkv.clone().requires_grad_(), table.clone().requires_grad_()
    both = torch.autograd.grad(F.rel_bias_attention(a, t, qc, kc, of, 2), [a, t], w)
    alone = (torch.autograd.grad(F.rel_bias_attention(a, table, qc, kc, of, 2), a, w)[0],
             torch.autograd.grad(F.rel_bias_attention(qkv, t, qc, kc, of, 2), t, w)[0])
    assert all(torch.equal(x, y) for x, y in zip(both, alone))
    q, kv = _rand(g, 3, 5, 128, device=dev), _rand(g, 3, 300, 256, device=dev)
    w = w[:, :5].contiguous()
    ql, kl = q.clone().requires_grad_(), kv.clone().requires_grad_()
    both = torch.autograd.grad(F.cross_attention(ql, kl, 2), [ql, kl], w)
    alone = (torch.autograd.grad(F.cross_attention(ql, kv, 2), ql, w)[0], torch.autograd.grad(F.cross_attention(q, kl, 2), kl, w)[0])
    assert all(torch.equal(x, y) for x, y in zip(both, alone))
    # no tokens at all
    e = torch.zeros(2, 0, 384, dtype=torch.bfloat16, device=dev, requires_grad=True)
    o = F.rel_bias_attention(e, t, qc[:0], kc[:0], of, 2)
    ge, gt = torch.autograd.grad(o, [e, t], torch.zeros_like(o))
    assert ge.shape == e.shape and not gt.any()


@gpu
def test_captured_answers():
    """Kernels with more than 64 KiB of LDS, split and joined, in a graph without gradients, replayed on new inputs."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(13)
    q, kv = _rand(g, 2, 1, 1024, device=dev), _rand(g, 2, 2000, 512, device=dev)
    lens = torch.tensor([2000, 3], dtype=torch.int32, device=dev)
    qc, kc, of = (t.to(dev) for t in _log(300, 64, 32))
    qkv, table = _rand(g, 1, 300, 768, device=dev), _rand(g, 32, 2, dtype=torch.float32, device=dev)

    @torch.no_grad()
    def answer():
        return F.cross_attention(q, kv, 8, 2, lens), F.rel_bias_attention(qkv, table, qc, kc, of, 2)

    answer()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = answer()
    for n in (3, 2000, 0, 777):
        lens[1] = n
        for t in (q, kv, qkv, table):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        want = answer()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))


@gpu
def test_captured_training_step_of_a_vit_with_options():
    from pytorch_distributed_training_amd import dist as pdist
    from pytorch_distributed_training_amd.engine import Engine, EngineConfig

    import os

    _dev("cuda")
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29541")
    pdist.init_process_group(backend="rccl", local_rank=0)
    g = torch.Generator().manual_seed(0)
    xs = [torch.rand(8, 3, 32, 32, generator=g).cuda() for _ in range(6)]
    ys = [torch.randint(0, 10, (8,), generator=g).cuda() for _ in range(6)]
    runs = []
    for graph in (False, True):
        eng = Engine(EngineConfig(model="vit_tiny_test", num_classes=10, optimizer="adamw", lr=1e-3, sync_bn=False, seed=0, graph=graph,
                                  model_options=OPTIONS))
        eng.optimizer.set_capturable(True)
        losses = [float(eng.train_step(x, y)) for x, y in zip(xs, ys)]
        assert not graph or eng._graph is not None, eng._graph_failed
        runs.append((losses, [p.detach().clone() for p in eng.net.parameters()]))
    assert runs[0][0] == runs[1][0]  # the same kernels on the same numbers, sums in a fixed order
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


@gpu
@pytest.mark.parametrize("case", [dict(b=512, nq=1, nk=197, heads=12, kv_heads=12, hd=64),
                                  dict(b=2, nq=3, nk=40000, heads=8, kv_heads=8, hd=128, lengths=[40000, 777], poison=True)],
                         ids=["pool", "long"])
def test_cross_attention_past_the_caches(case):
    """Keys and values of more than 256 MB: the variants that stream past the caches."""
    assert 4 * case["b"] * case["nk"] * case["kv_heads"] * case["hd"] >= 256 << 20
    _check_cross(_dev("cuda"), **case)


@gpu
@pytest.mark.parametrize("per_sample,post", [(True, False), (False, True)])
def test_gated_residual_norm_past_the_caches(per_sample, post):
    """Activations of more than 64 MB."""
    assert 64 * 530 * 1024 * 2 >= 64 << 20
    _check_norm(_dev("cuda"), (64, 530, 1024), per_sample, post, 0.5)


# ------------------------------------------------------------- rows whose every key has a very large negative bias
LARGE = [dict(b=1, n=40, hd=64), dict(b=2, n=70, hd=32), dict(b=1, n=150, hd=128), dict(b=1, n=600, hd=64), dict(b=3, n=300, hd=128)]


def _half_masked(n):
    """Codes that put the first half of the queries on bucket 1 for every key, the others on bucket 0."""
    q = torch.zeros(n, dtype=torch.int32)
    q[:n // 2] = 1
    return q, torch.zeros(n, dtype=torch.int32), torch.arange(2, dtype=torch.int32)


@gpu
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e9, -1e6, -8e3])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"b{c['b']}-n{c['n']}x{c['hd']}")
def test_rel_bias_backward_has_the_forward_weights(case, low):
    """V that names the first hd keys and dO that names the first hd queries show P in the output and in dV: one softmax."""
    dev = _dev("cuda")
    b, n, hd = case["b"], case["n"], case["hd"]
    m = min(n, hd)
    g = torch.Generator().manual_seed(31)
    qkv = _rand(g, b, n, 2, 3 * hd).view(b, n, 3, 2, hd)
    qkv[:, :, 2] = torch.eye(n, hd)[:, None]
    do = torch.eye(n, hd)[:, None].expand(b, n, 2, hd).reshape(b, n, 2 * hd).to(torch.bfloat16).to(dev)
    qkv = qkv.reshape(b, n, 6 * hd).to(dev).requires_grad_()
    table = torch.tensor([[0.3, -0.2], [low, 0.5]], device=dev)
    out = F.rel_bias_attention(qkv, table, *(t.to(dev) for t in _half_masked(n)), 2)
    (dqkv,) = torch.autograd.grad(out, qkv, do)
    forward = out.detach().view(b, n, 2, hd)[:, :m, :, :m].double()  # [b, query, head, key]
    backward = dqkv[..., 4 * hd:].view(b, n, 2, hd)[:, :m, :, :m].double().transpose(1, 3)
    # each of the two rounds P once and its result once; the scores of the two differ by roundings in 32 bits, which P takes up to
    # 2^-9 of (|bias| sqrt(hd) at most 2^16 has steps of 2^-8, half of it at each of hd / 16 additions, times 1 / sqrt(hd))
    _within(backward, forward, (4 * U + 2.0 ** -9 + hd / 16 * 2.0 ** -9 / math.sqrt(hd)) * forward + SLACK / n, "P")


@gpu
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e9])
@pytest.mark.parametrize("case", LARGE, ids=lambda c: f"b{c['b']}-n{c['n']}x{c['hd']}")
def test_rel_bias_gradients_of_absorbed_scores(case, low):
    """Where a bias takes up all of q . k a row's keys weigh the same, in every gradient too."""
    dev = _dev("cuda")
    heads, n, hd, b = 2, case["n"], case["hd"], case["b"]
    codes = _half_masked(n)
    table = torch.tensor([[0.3, -0.2], [low, 0.5]])
    qkv, table, qc, kc, of, do, live, (qkv64, do64) = _rel_case(dev, b, codes, heads, hd, table=table)
    leaf, tleaf = qkv.clone().requires_grad_(), table.clone().requires_grad_()
    out = F.rel_bias_attention(leaf, tleaf, qc, kc, of, heads)
    dqkv, dtable = torch.autograd.grad(out, [leaf, tleaf], do)
    q, k, v = qkv64.view(b, n, 3, heads, hd).permute(2, 0, 3, 1, 4)
    bias = table.double()[of.long()[(qc - kc[0]).long()]].t()[None, :, :, None].expand(b, heads, n, n).clone()
    gone = slice(0, n // 2)
    bias[:, 0, gone] = -(q[:, 0, gone] @ k[:, 0].transpose(-1, -2)) * hd ** -0.5  # the scores are nothing beside `low`
    do4 = do64.view(b, n, heads, hd).transpose(1, 2)
    (o, dq, dk, dv, ds, p), es = _attention64(q, k, v, bias, live, live.double(), do4)

    def flat(t):
        return t.transpose(1, 2).reshape(b, n, heads * hd)

    _within(out, flat(o), flat(es[0]), "out")
    for i, (name, w, e) in enumerate((("dq", dq, es[1]), ("dk", dk, es[2]), ("dv", dv, es[3]))):
        _within(dqkv[..., i * heads * hd:(i + 1) * heads * hd], flat(w), flat(e), name)
    # a bucket holds all pairs of its rows, whose dS add up to nothing; the bound is that of `_check_rel`
    err = p * (2.0 ** -15 * (do4.abs() * (o.abs() + p @ v.abs())).sum(-1, keepdim=True) + SLACK / 8 * (do4.abs() @ v.abs().transpose(-1, -2)))
    by_row = (err + 2.0 ** -20 * ds.abs()).sum((0, 3)), ds.sum((0, 3))
    bound, want = (torch.stack([t[:, n // 2:].sum(1), t[:, :n // 2].sum(1)]) for t in by_row)
    _within(dtable, want, bound, "dtable")


# ----------------------------------------------------------------------- what autograd has beyond a backward pass
def _three_calls(dev, seed=41):
    """-> (name, call, tensors that may get a tangent or a gradient): small calls that the kernels take"""
    g = torch.Generator().manual_seed(seed)
    qc, kc, of = (t.to(dev) for t in _log(9))
    qkv, q, kv = (_rand(g, 2, 9, w, device=dev) for w in (192, 64, 128))
    table, gate = (_rand(g, *s, dtype=torch.float32, device=dev) for s in ((8, 1), (64,)))
    one = torch.ones(64, device=dev)
    return [("rel_bias_attention", lambda a, b: F.rel_bias_attention(a, b, qc, kc, of, 1), [qkv, table]),
            ("cross_attention", lambda a, b: F.cross_attention(a, b, 1), [q, kv]),
            ("gated_residual_norm", lambda a, b: F.gated_residual_norm(a, a * 0.5, b, one, one)[1], [q, gate])]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_is_refused(device):
    """A tangent that the kernels would drop reads as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    for name, call, inputs in _three_calls(_dev(device)):
        for i in range(2):
            for grad in (False, True):
                with fwd.dual_level(), torch.set_grad_enabled(grad):
                    args = [t.clone().requires_grad_(grad) for t in inputs]
                    args[i] = fwd.make_dual(args[i], torch.ones_like(args[i]))
                    with pytest.raises((RuntimeError, NotImplementedError)):
                        call(*args)
        # a tangent that reaches the backward pass alone, from a later layer's weight
        args = [t.clone().requires_grad_() for t in inputs]
        with fwd.dual_level():
            out = call(*args)
            w = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            if device == "cuda":
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch.autograd.grad((out * w).sum(), args)
            else:  # elementary operations: the backward pass is linear in w
                got = fwd.unpack_dual(torch.autograd.grad((out * w).sum(), args)[0])
                assert got.tangent is not None and torch.equal(got.tangent, got.primal)


@pytest.mark.skipif(not pdt.native_available(), reason="extension not built")
def test_fake_tensors_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode

    for inside in (True, False):
        mode = FakeTensorMode()
        with mode:
            def e(*s, dtype=torch.bfloat16):
                return torch.empty(*s, dtype=dtype, device="cuda")
            qkv, q, kv, table, gate = e(2, 9, 192), e(2, 9, 64), e(2, 9, 128), e(8, 1, dtype=torch.float32), e(64, dtype=torch.float32)
            codes = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (9, 9, 33)]
            calls = [lambda: F.rel_bias_attention(qkv, table, *codes, 1), lambda: F.cross_attention(q, kv, 1),
                     lambda: F.gated_residual_norm(q, q, gate, gate, gate)]
            if inside:
                for call in calls:
                    with pytest.raises(RuntimeError, match="fake"):
                        call()
        if not inside:
            for call in calls:
                with pytest.raises(RuntimeError):
                    call()


@gpu
def test_tracers_and_transforms_are_refused():
    """They see only the allocation of the outputs; what they recorded would return memory that nobody has written."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    for name, call, (a, b) in _three_calls(_dev("cuda")):
        want = call(a, b)
        for grad in (False, True):
            x, y = a.clone().requires_grad_(grad), b.clone().requires_grad_(grad)
            for record in (lambda: torch.jit.trace(call, (x, y)), lambda: make_fx(call)(x, y), lambda: make_fx(call, pre_dispatch=True)(x, y),
                           lambda: make_fx(call, tracing_mode="fake")(x, y)):
                with pytest.raises(RuntimeError, match="cannot be traced"):
                    record()
            with pytest.raises(RuntimeError):
                torch.func.vmap(lambda t: call(t, y))(torch.stack([x, x]))
            with pytest.raises(RuntimeError):
                torch.func.grad(lambda t: call(t, y).float().sum())(x)
        # what only looks on, or leaves the calls out of what it records, works
        with FlopCounterMode(display=False):
            assert torch.equal(call(a, b), want)
        assert torch.equal(torch.compile(call, backend="eager")(a, b), want)


@pytest.mark.skipif(not pdt.native_available(), reason="extension not built")
def test_wrappers_without_memory_are_refused():
    """A subclass may say that it is on the GPU and hold its data elsewhere; its address is null."""
    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, *shape, dtype=torch.bfloat16):
            return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda")

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise AssertionError("the call was not refused before its first operation")

    f32, i32 = torch.float32, torch.int32
    qkv, q, kv, table, gate = Wrapper(2, 9, 192), Wrapper(2, 9, 64), Wrapper(2, 9, 128), Wrapper(8, 1, dtype=f32), Wrapper(64, dtype=f32)
    codes = [Wrapper(n, dtype=i32) for n in (9, 9, 33)]
    for call in (lambda: F.rel_bias_attention(qkv, table, *codes, 1), lambda: F.cross_attention(q, kv, 1),
                 lambda: F.cross_attention(q, kv, 1, lengths=Wrapper(2, dtype=i32)), lambda: F.gated_residual_norm(q, q, gate, gate, gate)):
        with pytest.raises(RuntimeError, match="memory of their own"):
            call()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_create_graph_raises_only_for_a_second_derivative(device):
    dev = _dev(device)
    for name, call, (a, b) in _three_calls(dev):
        x, y = a.clone().requires_grad_(), b.clone().requires_grad_()
        z = torch.full((3,), 0.5, device=dev, requires_grad=True)

        def loss():
            out = call(x, y)
            return (out * out).float().sum() + (z ** 3).sum()

        want = torch.autograd.grad(loss(), [x, y, z])
        got = torch.autograd.grad(loss(), [x, y, z], create_graph=True)
        assert all(torch.equal(u, v) for u, v in zip(want, got))
        (second,) = torch.autograd.grad(got[2].square().sum(), z)  # another term's
        assert torch.equal(second, 36 * z.detach() ** 3)
        for ask in (lambda d: torch.autograd.grad(d.float().sum(), x), lambda d: torch.autograd.grad(d.float().sum(), [x, y], allow_unused=True),
                    lambda d: (d.float().sum() + z.sum()).backward()):
            for i in (0, 1):
                got = torch.autograd.grad(loss(), [x, y], create_graph=True)
                with pytest.raises(RuntimeError):
                    ask(got[i])


def _check_codes(qkv, table, q, k, of):
    """The output for 64-bit codes against the plain form (codes are clamped where their differences would not fit)."""
    dev, (b, n, _), heads = qkv.device, qkv.shape, table.shape[1]
    out = F.rel_bias_attention(qkv, table, q, k, of, heads)
    limit = 2 ** 62 + 2 ** 28
    bucket = of[(q.clamp(-limit, limit)[:, None] - k.clamp(-limit, limit)[None]).clamp(0, of.numel() - 1)]
    x, y, v = qkv.double().view(b, n, 3, heads, -1).permute(2, 0, 3, 1, 4)
    live = _live(None, b, n, dev)
    (o, *_), (e, *_) = _attention64(x, y, v, table.double()[bucket].permute(2, 0, 1), live, live.double(), torch.zeros_like(x))
    _within(out, o.transpose(1, 2).reshape(out.shape), e.transpose(1, 2).reshape(out.shape), "out")


@gpu
@pytest.mark.parametrize("base", [2 ** 27, 2 ** 27 - 80, -2 ** 27 - 80, 2 ** 31 - 400, -2 ** 31, 1_765_000_000_000, -2 ** 62])
def test_rel_bias_codes_of_any_size(base):
    """Only differences count: positions that count from far away (clocks) give the bits of those that count from zero."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(43)
    qc, kc, of = (t.to(dev).long() for t in _log(150))
    qkv, w = _rand(g, 2, 150, 384, device=dev), _rand(g, 2, 150, 128, device=dev)
    table = _rand(g, 8, 2, dtype=torch.float32, device=dev)

    def run(q, k):
        a, t = qkv.clone().requires_grad_(), table.clone().requires_grad_()
        out = F.rel_bias_attention(a, t, q, k, of, 2)
        return (out, *torch.autograd.grad(out, [a, t], w))

    want = run(qc, kc)
    assert all(torch.equal(x, y) for x, y in zip(want, run(qc.int(), kc)))
    q, k = qc + base, kc + base
    forms = [(q, k)]
    if abs(base) < 2 ** 31 or base == -2 ** 31:
        forms += [(q.int(), k.int()), (q, k.int()), (q.int(), k)] if q.max() < 2 ** 31 else []
    for f in forms:
        assert all(torch.equal(x, y) for x, y in zip(want, run(*f)))
    strided = torch.stack([q, q + 1], 1)[:, 0]
    assert all(torch.equal(x, y) for x, y in zip(want, run(strided, k)))
    # one token far from the others, among the keys, among the queries; in both: no number at all
    step = 2 ** 27 if base > 0 else -2 ** 27
    q2, k2 = q.clone(), k.clone()
    q2[-1] += step
    k2[-1] += step
    _check_codes(qkv, table, q, k2, of)
    _check_codes(qkv, table, q2, k, of)
    out, dqkv, dtable = run(q2, k2)
    assert out.isnan().all() and dqkv.isnan().all() and dtable.isnan().any()  # (a bucket that no pair falls on keeps its zero)


@gpu
@pytest.mark.parametrize("base", [0, 2 ** 40])
@pytest.mark.parametrize("marks", [(2 ** 31 - 1, None), (None, -2 ** 31), (-2 ** 40, -2 ** 40), (-2 ** 63, 5), (2 ** 27, -2 ** 27 - 1), (-2 ** 27, 2 ** 27)], ids=str)
def test_rel_bias_marked_codes(marks, base):
    """Tokens marked by codes far from all others, on one axis or both: past the table's reach, and next to one another."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(89)
    qc, kc, of = (t.to(dev).long() for t in _log(90))
    qkv, table = _rand(g, 2, 90, 384, device=dev), _rand(g, 8, 2, dtype=torch.float32, device=dev)
    q, k = qc + base, kc + base
    for t, mark in ((q, marks[0]), (k, marks[1])):
        if mark is not None:
            t[:5] = mark
    if base and any(m is not None and 2 ** 27 <= m for m in marks):
        # (a mark of 2^27 or more is where that side's distances count from: 2^40 is too far from it for queries and keys)
        assert F.rel_bias_attention(qkv, table, q, k, of, 2).isnan().all()
    else:
        _check_codes(qkv, table, q, k, of)


@gpu
@pytest.mark.parametrize("case", [dict(b=1, n=600, heads=2), dict(b=2, n=300, heads=2), dict(b=1, n=1100, heads=1)], ids=lambda c: f"b{c['b']}-n{c['n']}-h{c['heads']}")
def test_rel_bias_table_gradient_at_large_scores(case):
    """Scores of some 500, launches whole and split: the weights of the backward add up to 1, not to what the rounding of
    log2(e) * maximum makes of them.  q . k is the same for all pairs and the bias grows towards the query's own position, so
    that all rows have one maximum (and one rounding, which would not average out), and parts of the keys have smaller ones."""
    dev = _dev("cuda")
    b, n, heads, hd = case["b"], case["n"], case["heads"], 64
    c = torch.tensor(math.log2(math.e) / 8, dtype=torch.float32)

    def off(t):  # of the exponents' base where the maximum is (512 + t) * 8
        m = torch.tensor((512 + t) * 8, dtype=torch.float32)
        return float(c.double() * m.double() - (c * m).double())

    steps = [max((k / 16 + 0.25 * j for j in range(4)), key=lambda t: abs(off(t))) for k in range(0, 128, 16)]  # one of each unit
    assert max(abs(off(t)) for t in steps) > 2.0 ** -16
    qc, kc, of = (t.to(dev) for t in _log(n))
    near = torch.zeros(8)  # buckets of _log: 0 the same place, 1 to 3 behind it, 4 (never), 5 to 7 ahead
    near[[0, 1, 2, 3, 5, 6, 7]] = torch.tensor([steps[7], steps[5], steps[3], steps[1], steps[6], steps[4], steps[2]])
    table = near[:, None].repeat(1, heads).to(dev).requires_grad_()
    qkv = torch.zeros(b, n, 3, heads, hd)
    qkv[:, :, :2, :, 0] = 64  # 512 of every score
    turn = torch.arange(n) * (math.pi / 24)  # dP = cos of the distance: near pairs and far ones get dS of one sign each
    wave = torch.stack([turn.cos(), turn.sin()], -1)[None, :, None]
    qkv[:, :, 2, :, :2] = wave
    do = torch.zeros(b, n, heads, hd)
    do[..., :2] = wave
    flat, do = (t.reshape(b, n, -1).to(torch.bfloat16).to(dev) for t in (qkv, do))
    out = F.rel_bias_attention(flat, table, qc, kc, of, heads)
    (got,) = torch.autograd.grad(out, table, do)
    q, k, v = flat.double().view(b, n, 3, heads, hd).permute(2, 0, 3, 1, 4)
    bucket = of.long()[(qc.long()[:, None] - kc.long()[None]).clamp(0, of.numel() - 1)]
    s = q @ k.transpose(-1, -2) * hd ** -0.5 + table.detach().double()[bucket].permute(2, 0, 1)
    p = torch.softmax(s, -1)
    do4 = do.double().view(b, n, heads, hd).transpose(1, 2)
    dp = do4 @ v.transpose(-1, -2)
    d = (p * dp).sum(-1, keepdim=True)

    def by_bucket(t):
        z = torch.zeros(8, heads, dtype=torch.float64, device=dev)
        return z.index_add_(0, bucket.reshape(-1), t.sum(0).reshape(heads, -1).t().contiguous())

    # the scores are exact (multiples of 2^-4 below 2^10).  P: an exponential (2^-23), a logarithm (of a sum below 2^11: 11 * 2^-24)
    # and c (2^-25 of an exponent below 2^4); dP has two terms; a sum over up to 2^11 keys, 2^6 sequential additions: 2^-20 covers them
    err = 2.0 ** -20 * p * (dp.abs() + d.abs() + 2)
    _within(got, by_bucket(p * (dp - d)), by_bucket(err), "dtable")


@gpu
@pytest.mark.parametrize("case", [dict(nq=1, nk=200), dict(nq=1, nk=3000), dict(nq=40, nk=200), dict(nq=40, nk=1500)], ids=lambda c: f"{c['nq']}x{c['nk']}")
def test_cross_attention_scores_of_minus_infinity(case):
    """Keys with an infinite channel whose scores are -inf weigh nothing, whole tiles of them too; all keys so: zeros."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(53)
    nq, nk, heads, hd = case["nq"], case["nk"], 2, 64
    q, kv = _rand(g, 2, nq, heads * hd, device=dev), _rand(g, 2, nk, 2 * heads * hd, device=dev)
    q.view(2, nq, heads, hd)[..., 0] = 1
    key0 = kv.view(2, nk, 2, heads, hd)[:, :, 0, :, 0]
    key0[0, :nk - 40] = -math.inf
    key0[0, 100:110] = 0.5
    key0[1] = -math.inf
    out = F.cross_attention(q, kv, heads)
    live = (key0[0, :, 0] > -math.inf).expand(2, nk)
    q4 = q.double().view(2, nq, heads, hd).transpose(1, 2)
    k4, v4 = kv.double().view(2, nk, 2, heads, hd).permute(2, 0, 3, 1, 4)
    k4 = k4.nan_to_num(neginf=0.0)
    (o, *_), (e, *_) = _attention64(q4, k4, v4, None, live, torch.ones(2, nq, device=dev).double(), torch.zeros_like(q4))
    _within(out[:1], o[:1].transpose(1, 2).reshape(1, nq, -1), e[:1].transpose(1, 2).reshape(1, nq, -1), "out")
    assert not out[1].any()


@gpu
def test_gated_residual_norm_with_a_gate_for_each_of_many_rows():
    dev = _dev("cuda")
    n, d = (1 << 23) + 1, 4
    x = torch.randn(n, d, device=dev, generator=torch.Generator(dev).manual_seed(59)).to(torch.bfloat16).requires_grad_()
    y = x.detach().flip(0).requires_grad_()
    gate = torch.linspace(-1, 1, n, device=dev)[:, None].repeat(1, d).requires_grad_()
    w, b = torch.full((d,), 1.5, device=dev, requires_grad=True), torch.zeros(d, device=dev, requires_grad=True)
    u, normed = F.gated_residual_norm(x, y, gate, w, b)
    got = torch.autograd.grad(u, [x, y, gate], torch.ones_like(u), retain_graph=True)
    assert torch.equal(got[0], torch.ones_like(x)) and torch.equal(got[1], gate.to(torch.bfloat16)) and torch.equal(got[2], y.float())
    (db,) = torch.autograd.grad(normed, b, torch.ones_like(normed))
    assert ((db - n).abs() <= 2.0 ** -10 * n).all()  # 2^14 rows a workgroup in one 32-bit sum each, all terms 1
    # the last rows of all against the form in 64 bits
    last = slice(n - 5, n)
    u64 = x[last].double() + gate[last].double() * y[last].double()
    n64 = torch.nn.functional.layer_norm(u64, (d,), w.double(), b.double(), 1e-6).detach()
    # (four channels: 2^-20 of what a division by a deviation of at least 2^-6 leaves)
    assert (n64 - normed[last].double()).abs().max() <= U * n64.abs().max() + 2.0 ** -14


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_gated_residual_norm_with_a_gate_for_each_row(device):
    """``x`` of two dimensions: the gate's first is the rows."""
    _check_norm(_dev(device), (37, 64), True, True, 0.5)
    _check_norm(_dev(device), (37, 64), True, False, 1.0)


def test_gated_residual_norm_oracle_with_a_gate_for_each_row_against_differences():
    g = torch.Generator().manual_seed(61)
    x, y, gate, w, b, pw, pb = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((3, 8),) * 3 + ((8,),) * 4)
    assert torch.autograd.gradcheck(lambda *t: F.gated_residual_norm(*t[:5], 1e-6, *t[5:], 0.5), (x, y, gate, w, b, pw, pb))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_no_sequences_no_queries_no_keys(device):
    dev = _dev(device)
    g = torch.Generator().manual_seed(67)

    def leaf(*s, dtype=torch.bfloat16):
        return _rand(g, *s, dtype=dtype, device=dev).requires_grad_()

    for b, nq, nk in ((0, 3, 4), (2, 0, 4), (2, 3, 0), (0, 0, 0), (2, 0, 0)):
        for lens in (None, torch.full((b,), 1, device=dev)):
            q, kv = leaf(b, nq, 128), leaf(b, nk, 128)
            out = F.cross_attention(q, kv, 4, 2, lens)
            got = torch.autograd.grad(out, [q, kv], torch.ones_like(out))
            assert out.shape == q.shape and got[0].shape == q.shape and got[1].shape == kv.shape
            assert not any(t.any() for t in (out, *got) if nk == 0 or nq == 0)
    for b, n in ((0, 3), (2, 0), (0, 0)):
        for lens in (None, torch.full((b,), 1, device=dev)):
            qkv, table = leaf(b, n, 192), leaf(8, 2, dtype=torch.float32)
            out = F.rel_bias_attention(qkv, table, *(t.to(dev) for t in _log(n)), 2, lens)
            got = torch.autograd.grad(out, [qkv, table], torch.ones_like(out))
            assert out.shape == (b, n, 64) and got[0].shape == qkv.shape and got[1].shape == table.shape and not got[1].any()
    for shape in ((0, 8), (0, 3, 8), (3, 0, 8)):
        for gate in (leaf(8, dtype=torch.float32), leaf(shape[0], 8, dtype=torch.float32)):
            x, w = leaf(*shape), leaf(8, dtype=torch.float32)
            new, normed = F.gated_residual_norm(x, x, gate, w, w, 1e-6, w, w)
            got = torch.autograd.grad([new, normed], [x, gate, w], [torch.ones_like(x)] * 2)
            assert new.shape == normed.shape == x.shape and got[0].shape == x.shape and got[1].shape == gate.shape
            assert not any(t.any() for t in got)


@gpu
@pytest.mark.parametrize("case", [dict(n=4000, heads=17, far=2047), dict(n=4200, heads=16, far=16), dict(n=16500, heads=1, far=16),
                                  dict(n=16500, heads=2, far=16)], ids=lambda c: f"n{c['n']}-h{c['heads']}-far{c['far']}")
def test_rel_bias_table_gradient_in_groups(case):
    """More than 1 GiB of sums over pairs: groups of heads (16 + 1, 15 + 1) and blocks of queries (127 + 2 of 128), each both with
    the far pairs summed by the dQ pass (more positions than entries, dQ in one part) and without."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(71)
    n, heads, hd = case["n"], case["heads"], 32
    qc, kc, of = (t.to(dev) for t in _log(n, case["far"], 8))
    qkv, do = _rand(g, 1, n, 3 * heads * hd, device=dev), _rand(g, 1, n, heads * hd, std=0.1, device=dev)
    table = _rand(g, 8, heads, dtype=torch.float32, device=dev).requires_grad_()
    out = F.rel_bias_attention(qkv, table, qc, kc, of, heads)
    (got,) = torch.autograd.grad(out, table, do)
    want, bound = (torch.zeros(8, heads, dtype=torch.float64, device=dev) for _ in range(2))
    for h in range(heads):
        q, k, v = qkv.view(n, 3, heads, hd)[:, :, h].double().unbind(1)
        w = do.view(n, heads, hd)[:, h].double()
        for rows in torch.arange(n, device=dev).split(2048):
            bucket = of.long()[(qc[rows, None] - kc[None]).clamp(0, of.numel() - 1).long()]
            p = torch.softmax(q[rows] @ k.t() * hd ** -0.5 + table.detach()[bucket, h].double(), -1)
            o, dp, x = p @ v, w[rows] @ v.t(), w[rows]
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            # the bound of `_check_rel`
            err = p * (2.0 ** -15 * (x.abs() * (o.abs() + p @ v.abs())).sum(-1, keepdim=True) + SLACK / 8 * (x.abs() @ v.abs().t()))
            err += 2.0 ** -20 * ds.abs()
            for i in range(8):
                here = (bucket == i).double()
                want[i, h] += (ds * here).sum()
                bound[i, h] += (err * here).sum()
    _within(got, want, bound, "dtable")


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("n", [1, 45, 300])
def test_unidirectional_buckets_for_a_decoder(device, n):
    """As its documentation has it: later keys in a bucket of their own whose row is -inf."""
    dev = _dev(device)
    g = torch.Generator().manual_seed(73)
    heads, hd, buckets, far = 2, 32, 8, 20
    qc, kc, of = pdt.nn.log_position_buckets(n, buckets, far, bidirectional=False)
    of[:far] = buckets
    qc, kc, of = (t.to(dev) for t in (qc, kc, of))
    qkv, do = _rand(g, 2, n, 3 * heads * hd, device=dev).requires_grad_(), _rand(g, 2, n, heads * hd, std=0.1, device=dev)
    learned = _rand(g, buckets, heads, dtype=torch.float32, device=dev).requires_grad_()
    table = torch.cat([learned, learned.new_full((1, heads), -math.inf)])
    out = F.rel_bias_attention(qkv, table, qc, kc, of, heads)
    dqkv, dtable = torch.autograd.grad(out, [qkv, learned], do)
    q, k, v = qkv.detach().double().view(2, n, 3, heads, hd).permute(2, 0, 3, 1, 4)
    i = torch.arange(n, device=dev)
    near = (i[:, None] - i[None]).clamp(min=0)
    bucket = of.long()[(near + far).clamp(max=2 * far)]
    bias = learned.detach().double()[bucket].permute(2, 0, 1).masked_fill(i[None] > i[:, None], -math.inf)
    do4 = do.double().view(2, n, heads, hd).transpose(1, 2)
    one = torch.ones(2, n, device=dev)
    (o, dq, dk, dv, ds, _), es = _attention64(q, k, v, bias, one.bool(), one.double(), do4)
    for i, (got, w, e) in enumerate(zip((out, *dqkv.split(heads * hd, -1)), (o, dq, dk, dv), es)):
        _within(got, w.transpose(1, 2).reshape(2, n, -1), e.transpose(1, 2).reshape(2, n, -1), ("out", "dq", "dk", "dv")[i])
    assert torch.isfinite(dtable).all()


@gpu
def test_capture_beside_an_eager_graph_of_leaves_behind_the_inputs_is_refused():
    """Parameters that are cast and expanded before the call (an attention pool's query) are leaves of its backward pass too."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(79)
    qc, kc, of = (t.to(dev) for t in _log(9))
    table, q, gate = (_rand(g, *s, dtype=torch.float32, device=dev).requires_grad_() for s in ((4, 1), (1, 1, 64), (64,)))
    qkv, kv, x = (_rand(g, 2, 9, w, device=dev) for w in (192, 128, 64))
    one = torch.ones(64, device=dev)
    for call, leaf in ((lambda: F.rel_bias_attention(qkv, torch.cat([table, table * 0.5]), qc, kc, of, 1), table),
                       (lambda: F.cross_attention(q.to(torch.bfloat16).expand(2, -1, -1), kv, 1), q),
                       (lambda: F.gated_residual_norm(x, x, gate * 2, one, one)[0], gate)):
        alive = call()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                one * 2
                call()
        want = torch.autograd.grad(alive, leaf, torch.ones_like(alive))[0]
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
            (got,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        # an input computed before the capture: its gradient would go to the stream of its own node, outside
        y = leaf * 1.0
        late = {table: lambda: F.rel_bias_attention(qkv, torch.cat([y, y * 0.5]), qc, kc, of, 1),
                q: lambda: F.cross_attention(y.to(torch.bfloat16).expand(2, -1, -1), kv, 1),
                gate: lambda: F.gated_residual_norm(x, x, y, one, one)[0]}[leaf]
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                one * 2
                late()
        y = y.detach().requires_grad_()
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            late()


@gpu
def test_negated_views():
    """The imaginary part of a conjugate is a view of numbers that are yet to be negated."""
    dev = _dev("cuda")
    g = torch.Generator().manual_seed(83)

    def negated(t):
        v = torch.imag(torch.complex(torch.zeros_like(t), t).conj()) if t.dtype == torch.float32 else torch._neg_view(t)
        assert v.is_neg()
        return v

    x, w = _rand(g, 2, 9, 64, device=dev), _rand(g, 2, 9, 64, device=dev)
    v = _rand(g, 64, dtype=torch.float32, device=dev)
    for u, n in zip(F.gated_residual_norm(negated(x), x, negated(v), negated(v), v), F.gated_residual_norm(-x, x, -v, -v, v)):
        assert torch.equal(u, n)
    kv, lens = _rand(g, 2, 40, 128, device=dev), torch.tensor([-7, -40], device=dev, dtype=torch.int32)
    assert torch.equal(F.cross_attention(negated(x), negated(kv), 1, None, negated(lens)), F.cross_attention(-x, -kv, 1, None, -lens))
    qc, kc, of = (t.to(dev) for t in _log(40))
    qkv, table = _rand(g, 2, 40, 192, device=dev), _rand(g, 8, 1, dtype=torch.float32, device=dev)
    assert torch.equal(F.rel_bias_attention(negated(qkv), negated(table), negated(kc), negated(qc), of, 1),
                       F.rel_bias_attention(-qkv, -table, -kc, -qc, of, 1))
    q = x.clone().requires_grad_()
    for grad in (negated(w), torch._efficientzerotensor(w.shape, dtype=w.dtype, device=dev)):
        out = F.cross_attention(q, kv, 1)
        (a,) = torch.autograd.grad(out, q, grad, retain_graph=True)
        (b,) = torch.autograd.grad(out, q, grad + torch.zeros_like(w))
        assert torch.equal(a, b)


@gpu
def test_modes_around_the_calls():
    """Inference mode, checkpointing of both kinds and saved tensors that wait on the host give the bits of a plain call."""
    from torch.utils.checkpoint import checkpoint

    for name, call, inputs in _three_calls(_dev("cuda")):
        args = [t.clone().requires_grad_() for t in inputs]
        out = call(*args)
        w = torch.ones_like(out)
        w[:, 1::2] = -0.5
        want = torch.autograd.grad(out, args, w)
        with torch.inference_mode():
            assert torch.equal(call(*inputs), out)
            assert torch.equal(call(*(t.clone() for t in inputs)), out)
        with torch.no_grad():
            assert torch.equal(call(*args), out)
        for reentrant in (False, True):
            again = [t.clone().requires_grad_() for t in inputs]
            checkpoint(call, *again, use_reentrant=reentrant).backward(w)
            assert all(torch.equal(t.grad, g) for t, g in zip(again, want))
        with torch.autograd.graph.save_on_cpu(pin_memory=True):
            out = call(*args)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, args, w), want))
        # an input changed between the passes is an error, not a wrong gradient
        x = inputs[0].clone().requires_grad_()
        y = x * 1.0
        out = call(y, inputs[1])
        with torch.no_grad():
            y.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(out, x, w)


@gpu
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_rel_bias_masks_of_different_depth(hd):
    """Rows of several masking values only: the least low wins, as in the plain form, up to the ends of the type."""
    dev = _dev("cuda")
    lowest, low16 = torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min
    g = torch.Generator().manual_seed(97)
    n = 60
    qc, kc = torch.arange(n, dtype=torch.int32) % 5 * 100, -torch.arange(n, dtype=torch.int32) % 7  # an entry a pair of residues
    of = torch.randint(0, 4, (420,), generator=g)
    for values in ((lowest, -1e30, -1e30, lowest), (low16, lowest, low16, lowest), (-2e38, -3e38, -1e37, -1e36), (-math.inf, lowest, -math.inf, lowest),
                   (3e38, 1e38, -3e38, lowest)):
        table = torch.tensor(values)[:, None].repeat(1, 2)
        _check_rel(dev, 2, (qc, kc, of), 2, hd, table=table, seed=int(g.initial_seed()))
