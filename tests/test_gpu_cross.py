"""GPU: attention to an encoder's states of another length (dm_cross_fwd / dm_cross_bwd) against the definition in 64 bits.

Tolerances (u = 2^-24; ub = 2^-8 for bf16 operands, 0 for fp32), per element, from the reference's own intermediate values:
  score         ds = (hd + 4) u scale |q| |k|  (products and sums of a dot product) + 4 u (1 + |s| + |s - m|)  (the base-2
                argument of the exponential and the exponential itself);  a probability is off by a factor 1 +- e,
                e = 2 max(ds) + (Nk + 4) u  (its own score, the row sum), and by ub once more where it is rounded
  o             ub |o| + (e + ub + (Nk + 4) u) sum p |v|
  lse           max(ds) + (Nk + 8) u + 4 u |lse|
  dS            p [ddelta + (hd + 4) u |dO| |v|] + (e + ub) |dS|,  ddelta = sum |dO| tol(o) + (hd + 4) u sum |dO| |o|
  dq, dk, dv    ub |result| + the tolerance of dS (of p) through |k| (|q|, |dO|) + n u of the n-term sum of magnitudes
Everything is doubled once for second-order terms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


def K():
    from diffusion_model_amd import kernels
    return kernels


def valid_rows(c, Nk, lens, mask):
    if c is None:
        return torch.zeros(0, dtype=torch.long)
    n = Nk if lens is None else max(0, min(Nk, int(lens[c])))
    r = torch.arange(n)
    return r if mask is None else r[mask[c, :n].bool()]


def reference(q, k, v, heads, kv_heads, lens=None, mask=None, index=None, scale=None, d_o=None, keep=None):
    """Values and tolerances in 64 bits.  keep: optional [B, H, Nq, Nk] multiplier of the probabilities (dropout)."""
    ub = 2.0 ** -8 if q.dtype == BF16 else 0.0
    B, Nq, Cq = q.shape
    Bc, Nk, _ = k.shape
    hd = Cq // heads
    scale = hd ** -0.5 if scale is None else scale
    q, k, v = q.double(), k.double(), v.double()
    val = dict(o=torch.zeros_like(q), lse=torch.full((B, heads, Nq), -math.inf, dtype=torch.float64), dq=torch.zeros_like(q),
               dk=torch.zeros_like(k), dv=torch.zeros_like(k))
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    mag = dict(dk=torch.zeros_like(k), dv=torch.zeros_like(k))
    terms = torch.zeros(Bc)
    for b in range(B):
        c = (0 if Bc == 1 else b) if index is None else int(index[b])
        c = c if 0 <= c < Bc else None
        rows = valid_rows(c, Nk, lens, mask)
        if rows.numel() == 0:
            continue
        n = rows.numel()
        for h in range(heads):
            hs = slice(h * hd, (h + 1) * hd)
            gs = slice((h // (heads // kv_heads)) * hd, (h // (heads // kv_heads) + 1) * hd)
            qh, kh, vh = q[b, :, hs], k[c, rows][:, gs], v[c, rows][:, gs]
            s = qh @ kh.T * scale
            m = s.amax(-1, keepdim=True)
            lse = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - lse)
            z = torch.ones_like(p) if keep is None else keep[b, h][:, rows].double()
            err_s = (hd + 4) * U * scale * (qh.abs() @ kh.abs().T) + 4 * U * (1 + s.abs() + (s - m).abs())
            e = 2 * err_s.amax(-1, keepdim=True) + (n + 4) * U
            o = (p * z) @ vh
            t_o = ub * o.abs() + (e + ub + (n + 4) * U) * ((p * z) @ vh.abs())
            val["o"][b, :, hs], tol["o"][b, :, hs] = o, 2 * t_o
            val["lse"][b, h] = lse[:, 0]
            tol["lse"][b, h] = 2 * (err_s.amax(-1) + (n + 8) * U + 4 * U * lse[:, 0].abs())
            if d_o is None:
                continue
            g = d_o[b, :, hs].double()
            dp, delta = g @ vh.T * z, (g * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            t_delta = (g.abs() * t_o).sum(-1, keepdim=True) + (hd + 4) * U * (g.abs() * o.abs()).sum(-1, keepdim=True)
            t_ds = p * (t_delta + (hd + 4) * U * (g.abs() @ vh.abs().T) * z) + (e + ub) * ds.abs()
            t_p = (e + ub) * p * z
            val["dq"][b, :, hs] = ds @ kh * scale
            tol["dq"][b, :, hs] = 2 * (ub * val["dq"][b, :, hs].abs() + scale * ((t_ds + (n + 4) * U * ds.abs()) @ kh.abs()))
            for j, name, left, t_left, right in ((0, "dk", ds * scale, t_ds * scale, qh), (1, "dv", p * z, t_p, g)):
                full, t_full, m_full = (torch.zeros(Nk, hd, dtype=torch.float64) for _ in range(3))
                full[rows], t_full[rows], m_full[rows] = left.T @ right, t_left.T @ right.abs(), left.abs().T @ right.abs()
                val[name][c, :, gs] += full
                tol[name][c, :, gs] += t_full
                mag[name][c, :, gs] += m_full
            terms[c] += Nq
    for name in ("dk", "dv"):
        t = terms.double()[:, None, None]
        tol[name] = 2 * (tol[name] + (t + 8) * U * mag[name] + ub * val[name].abs())
    return val, tol


def check(name, got, val, tol):
    got, want, t = got.double().cpu(), val[name], tol[name]
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin]), name
    err = (got[fin] - want[fin]).abs()
    assert bool((err <= t[fin]).all()), f"{name}: worst excess {float((err - t[fin]).max()):.3e}, worst error {float(err.max()):.3e}"


def inputs(dtype, B, Bc, Nq, Nk, H, G, hd, lens, mask, index, seed=0, sharp=1.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    q, k, v, d_o = r(B, Nq, H * hd), r(Bc, Nk, G * hd), r(Bc, Nk, G * hd), r(B, Nq, H * hd)
    if sharp != 1.0:
        q = (q.float() * sharp).to(dtype)
    L = M = I = None
    if lens:
        L = torch.randint(0, Nk + 1, (Bc,), generator=g, dtype=torch.int32)
        L[0] = 0 if lens == "empty" else Nk
        if Bc > 1:
            L[1] = 1
    if mask:
        M = torch.rand(Bc, Nk, generator=g) < 0.7
        if Bc > 1:
            M[Bc - 1] = False
    if index:
        I = torch.randint(0, Bc, (B,), generator=g, dtype=torch.int32)
    return q, k, v, d_o, L, M, I


def poison(k, v, lens, mask):
    """NaN and infinities in every state that does not count."""
    k, v = k.clone(), v.clone()
    for c in range(k.shape[0]):
        bad = torch.ones(k.shape[1], dtype=torch.bool)
        bad[valid_rows(c, k.shape[1], lens, mask)] = False
        k[c, bad], v[c, bad] = float("nan"), float("inf")
    return k, v


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


CASES = [
    # B, Bc, Nq, Nk, H, G, hd, lens, mask, index
    (2, 2, 1, 1, 1, 1, 8, None, False, False),               # one query, one state
    (3, 3, 1, 700, 2, 1, 64, "ragged", False, False),        # one query, the keys split over workgroups
    (1, 1, 5, 2100, 2, 2, 40, None, True, False),            # few queries, long states, holes
    (4, 4, 33, 77, 4, 4, 32, "empty", False, False),         # one context without states
    (2, 2, 129, 64, 8, 8, 16, None, False, False),
    (3, 3, 100, 65, 2, 2, 24, "empty", True, False),         # lengths and holes together; one context masked whole
    (2, 2, 40, 31, 6, 2, 80, "ragged", False, False),        # heads shared by three
    (2, 2, 70, 300, 4, 1, 96, None, True, False),
    (2, 2, 65, 200, 2, 2, 128, "ragged", False, False),
    (1, 1, 260, 129, 3, 1, 104, None, False, False),
    (7, 3, 50, 45, 2, 2, 32, "ragged", False, True),         # samples share contexts
    (66, 2, 9, 20, 2, 1, 16, "ragged", True, True),          # more samples than one wave scans at a time
    (5, 1, 40, 33, 2, 2, 8, None, False, False),             # one context for all
    (2, 2, 17, 600, 2, 2, 128, "ragged", True, False),       # more keys than one image holds
    (2, 2, 64, 1500, 2, 1, 128, "ragged", True, False),      # two query tiles, two waves each
    (1, 1, 200, 900, 1, 1, 128, "ragged", False, False),     # streamed keys, split
    (1, 1, 20, 9000, 1, 1, 128, None, False, False),         # more keys than 64 images hold
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Bc,Nq,Nk,H,G,hd,lens,mask,index", CASES)
def test_cross_forward_and_backward(B, Bc, Nq, Nk, H, G, hd, lens, mask, index, dtype):
    kn = K()
    q, k, v, d_o, L, M, I = inputs(dtype, B, Bc, Nq, Nk, H, G, hd, lens, mask, index)
    val, tol = reference(q, k, v, H, G, L, M, I, d_o=d_o)
    kp, vp = poison(k, v, L, M)
    dq_, dk_, dv_, do_, dL, dM, dI = cuda(q, kp, vp, d_o, L, M, I)
    kw = dict(kv_heads=G, lens=dL, mask=dM, index=dI)
    o, lse = kn.cross_fwd(dq_, dk_, dv_, H, **kw)
    check("o", o, val, tol)
    check("lse", lse, val, tol)
    first = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    for name, t in zip(("dq", "dk", "dv"), first):
        check(name, t, val, tol)
    again = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, again))      # fixed summation order


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,H,G,hd,Nk,lens,mask,index", [
    (1, 2, 2, 8, 5, None, False, False), (1, 2, 2, 24, 300, "ragged", True, False), (1, 3, 3, 40, 1, None, False, False),
    (1, 4, 2, 64, 1500, "ragged", False, True), (2, 2, 2, 104, 600, "empty", False, False), (1, 4, 1, 128, 513, None, True, True),
    (3, 1, 1, 16, 257, "empty", True, False), (1, 3, 1, 80, 700, "ragged", False, False), (1, 2, 2, 64, 20000, "ragged", False, False)])
def test_cross_single_queries(Nq, H, G, hd, Nk, lens, mask, index, dtype):
    """Up to four rows on a key / value head take the streaming kernel, with and without key splits."""
    kn = K()
    q, k, v, d_o, L, M, I = inputs(dtype, 3, 3, Nq, Nk, H, G, hd, lens, mask, index, seed=Nk)
    val, tol = reference(q, k, v, H, G, L, M, I)
    kp, vp = poison(k, v, L, M)
    qd, kd, vd, Ld, Md, Id = cuda(q, kp, vp, L, M, I)
    o, lse = kn.cross_fwd(qd, kd, vd, H, kv_heads=G, lens=Ld, mask=Md, index=Id)
    assert kn.last_variant().startswith("cross_one")
    check("o", o, val, tol)
    check("lse", lse, val, tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_scale_and_large_scores(dtype):
    """A scale of the caller's, and scores far apart: the running maximum moves from block to block."""
    kn = K()
    q, k, v, d_o, *_ = inputs(dtype, 1, 1, 70, 400, 2, 2, 32, None, False, False, seed=3, sharp=6.0)
    val, tol = reference(q, k, v, 2, 2, scale=0.9, d_o=d_o)
    q, k, v, d_o = cuda(q, k, v, d_o)
    o, lse = kn.cross_fwd(q, k, v, 2, scale=0.9)
    check("o", o, val, tol)
    check("lse", lse, val, tol)
    for name, t in zip(("dq", "dk", "dv"), kn.cross_bwd(q, k, v, o, lse, d_o, 2, scale=0.9)):
        check(name, t, val, tol)


def test_cross_strided_views_and_untouched_neighbours():
    """k and v from one fused projection, q from a wider buffer, every result into a slice: the rest stays as it was."""
    kn = K()
    B, Nq, Nk, H, hd = 2, 50, 40, 4, 16
    C = H * hd
    q, k, v, d_o, L, _, _ = inputs(BF16, B, B, Nq, Nk, H, H, hd, "ragged", False, False, seed=5)
    val, tol = reference(q, k, v, H, H, L, d_o=d_o)
    big = torch.full((B, Nq, 3 * C), 7.0, dtype=BF16, device="cuda")
    big[..., C:2 * C] = q.cuda()
    kv = torch.cat([k, v], -1).cuda()
    ob, dqb = torch.full_like(big, 5.0), torch.full_like(big, 5.0)
    dkv = torch.full((B, Nk, 3 * C), 5.0, dtype=BF16, device="cuda")
    args = (big[..., C:2 * C], kv[..., :C], kv[..., C:])
    o, lse = kn.cross_fwd(*args, H, lens=L.cuda(), out=ob[..., C:2 * C])
    check("o", o, val, tol)
    dq, dk, dv = kn.cross_bwd(*args, o, lse, d_o.cuda(), H, lens=L.cuda(), dq=dqb[..., :C], dk=dkv[..., :C], dv=dkv[..., 2 * C:])
    for name, t in (("dq", dqb[..., :C]), ("dk", dkv[..., :C]), ("dv", dkv[..., 2 * C:])):
        check(name, t, val, tol)
    for rest in (ob[..., :C], ob[..., 2 * C:], dqb[..., C:], dkv[..., C:2 * C]):
        assert bool((rest == 5.0).all())


def test_cross_index_outside_the_contexts_and_odd_lengths():
    """An index outside [0, Bc) means no states; lengths outside [0, Nk] are clamped."""
    kn = K()
    q, k, v, d_o, *_ = inputs(F32, 5, 3, 20, 33, 2, 2, 16, None, False, False, seed=6)
    index = torch.tensor([2, -1, 0, 3, 2], dtype=torch.int32)
    lens = torch.tensor([100, 5, -7], dtype=torch.int32)
    val, tol = reference(q, k, v, 2, 2, lens, None, index, d_o=d_o)
    assert not bool(torch.isfinite(val["lse"][[0, 1, 3, 4]]).any()) and bool(torch.isfinite(val["lse"][2]).all())
    q, k, v, d_o, lens, index = cuda(q, k, v, d_o, lens, index)
    o, lse = kn.cross_fwd(q, k, v, 2, lens=lens, index=index)
    check("o", o, val, tol)
    check("lse", lse, val, tol)
    for name, t in zip(("dq", "dk", "dv"), kn.cross_bwd(q, k, v, o, lse, d_o, 2, lens=lens, index=index)):
        check(name, t, val, tol)


def test_cross_no_states_and_empty_batches():
    kn = K()
    q = torch.randn(2, 7, 32, device="cuda")
    k = torch.empty(2, 0, 32, device="cuda")
    o, lse = kn.cross_fwd(q, k, k, 2)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = kn.cross_bwd(q, k, k, o, lse, q, 2)
    assert bool((dq == 0).all()) and dk.shape == k.shape
    k = torch.randn(2, 5, 32, device="cuda")
    none = q[:, :0].contiguous()
    o, lse = kn.cross_fwd(none, k, k, 2)
    assert o.shape == (2, 0, 32) and lse.shape == (2, 2, 0)
    dq, dk, dv = kn.cross_bwd(none, k, k, o, lse, none, 2)
    assert bool((dk == 0).all()) and bool((dv == 0).all())


def test_cross_nan_in_a_valid_state_reaches_only_its_sample():
    kn = K()
    q, k, v, *_ = inputs(BF16, 2, 2, 40, 50, 2, 2, 32, None, False, False, seed=8)
    v[0, 3, 0] = float("nan")
    o, lse = kn.cross_fwd(*cuda(q, k, v), 2)
    assert bool(torch.isnan(o[0, :, 0]).all()) and bool(torch.isfinite(o[1]).all()) and bool(torch.isfinite(lse).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hd,Nk,Nq", [(128, 100, 150), (64, 50, 150), (128, 100, 20), (128, 100, 50), (64, 30, 40), (32, 20, 1)])
def test_cross_dropout(hd, Nk, Nq, dtype):
    """The keep mask is read off with unit values (o = P Z / keep), is a fair draw, and the same seed then gives the
    forward and the backward of exactly that mask."""
    kn = K()
    B, H, p = 2, 2, 0.25
    q, k, v, d_o, L, _, _ = inputs(dtype, B, B, Nq, Nk, H, H, hd, "ragged", False, False, seed=9)
    L[:] = Nk
    eye = torch.zeros(B, Nk, H, hd)
    eye[:, torch.arange(Nk), :, torch.arange(Nk)] = 1.0
    qd, kd, vd, dd, Ld = cuda(q, k, v, d_o, L)
    o, _ = kn.cross_fwd(qd, kd, eye.reshape(B, Nk, -1).to(dtype).cuda(), H, lens=Ld, drop_p=p, drop_seed=77)
    keep = (o.float().cpu().reshape(B, Nq, H, hd).permute(0, 2, 1, 3)[..., :Nk] > 0).double()
    n = keep.numel()
    assert abs(float(keep.mean()) - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n)       # five standard deviations
    keep = keep / (1.0 - round(p * 32768) / 32768)
    val, tol = reference(q, k, v, H, H, L, d_o=d_o, keep=keep)
    o, lse = kn.cross_fwd(qd, kd, vd, H, lens=Ld, drop_p=p, drop_seed=77)
    check("o", o, val, tol)
    check("lse", lse, val, tol)
    for name, t in zip(("dq", "dk", "dv"), kn.cross_bwd(qd, kd, vd, o, lse, dd, H, lens=Ld, drop_p=p, drop_seed=77)):
        check(name, t, val, tol)
    other, _ = kn.cross_fwd(qd, kd, vd, H, lens=Ld, drop_p=p, drop_seed=78)
    assert not torch.equal(other, o)


def test_cross_gradients_against_differences():
    """fp32, along random directions: (f(x + eps d) - f(x - eps d)) / 2 eps.  eps = 1e-2: the third-order term is about
    eps^2 / 6 of the directional derivative's scale, the roundings about |f| 2^-22 / eps."""
    kn = K()
    q, k, v, w, L, M, I = inputs(F32, 3, 2, 12, 20, 2, 1, 16, "ragged", True, True, seed=11)
    M[:] = True
    M[0, 4] = False
    dw, dL, dM, dI = cuda(w, L, M, I)
    kw = dict(kv_heads=1, lens=dL, mask=dM, index=dI)
    f = lambda a, b, c: float((kn.cross_fwd(a.cuda(), b.cuda(), c.cuda(), 2, **kw)[0].double() * dw.double()).sum())
    qd, kd, vd = cuda(q, k, v)
    o, lse = kn.cross_fwd(qd, kd, vd, 2, **kw)
    grads = [t.double().cpu() for t in kn.cross_bwd(qd, kd, vd, o, lse, dw, 2, **kw)]
    g = torch.Generator().manual_seed(12)
    for i in range(3):
        d = torch.randn((q, k, v)[i].shape, generator=g)
        eps = 1e-2
        hi, lo = [list((q, k, v)) for _ in range(2)]
        hi[i], lo[i] = hi[i] + eps * d, lo[i] - eps * d
        num = (f(*hi) - f(*lo)) / (2 * eps)
        want = float((grads[i] * d.double()).sum())
        size = float((grads[i].abs() * d.abs().double()).sum())
        assert abs(num - want) < 2e-3 * size + 1e-3, (i, num, want)


@pytest.mark.parametrize("shape", [(4, 2, 200, 70, 4, 2, 32), (2, 2, 3, 900, 2, 2, 64), (2, 2, 20, 900, 2, 2, 64), (2, 2, 80, 900, 2, 2, 64), (5, 2, 1, 400, 2, 2, 64)])
def test_cross_captured_replays(shape):
    """Forward and backward in one HIP graph, replayed with other inputs and other lengths, eager calls in between."""
    kn = K()
    B, Bc, Nq, Nk, H, G, hd = shape
    q, k, v, d_o, L, M, I = cuda(*inputs(BF16, *shape, "ragged", True, Bc != B))
    kw = dict(kv_heads=G, lens=L, mask=M, index=I)

    def step():
        o, lse = kn.cross_fwd(q, k, v, H, **kw)
        return (o, lse, *kn.cross_bwd(q, k, v, o, lse, d_o, H, **kw))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        fresh = cuda(*inputs(BF16, *shape, "empty" if i % 2 else "ragged", True, Bc != B, seed=20 + i))
        for t, n in zip((q, k, v, d_o, L, M, I), fresh):
            if t is not None:
                t.copy_(n)
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i


@pytest.mark.parametrize("Nq", [4, 20, 40])
def test_cross_two_streams_at_once(Nq):
    """Two calls that need scratch, on two streams, many times: each has its own."""
    kn = K()
    sets = [cuda(*inputs(BF16, 2, 2, Nq, 1500, 2, 2, 64, None, False, False, seed=s))[:4] for s in (1, 2)]

    def both(q, k, v, d_o):
        o, lse = kn.cross_fwd(q, k, v, 2)
        return (o, lse, *kn.cross_bwd(q, k, v, o, lse, d_o, 2))

    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(both(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for run in got[i] for a, b in zip(run, want[i]))


@pytest.mark.parametrize("Nq", [1, 20, 40])
def test_cross_states_past_32_bits(Nq):
    """Rows of k and v whose byte offsets pass 2^32."""
    kn = K()
    Nk, ld = 600, 1 << 22
    base = torch.empty(1, Nk, ld, dtype=BF16, device="cuda")      # 4.7 GiB
    q, k, v, d_o, *_ = inputs(BF16, 1, 1, Nq, Nk, 1, 1, 32, None, False, False, seed=13)
    kd, vd = base[..., :32], base[..., 64:96]
    kd.copy_(k)
    vd.copy_(v)
    val, tol = reference(q, k, v, 1, 1, d_o=d_o)
    qd, dd = cuda(q, d_o)
    o, lse = kn.cross_fwd(qd, kd, vd, 1)
    check("o", o, val, tol)
    for name, t in zip(("dq", "dk", "dv"), kn.cross_bwd(qd, kd, vd, o, lse, dd, 1, dk=base[..., 128:160], dv=base[..., 192:224])):
        check(name, t, val, tol)


def test_cross_refuses_outputs_that_are_operands():
    q, k, v = (torch.zeros(2, n, 32, dtype=BF16, device="cuda") for n in (5, 7, 7))
    for t in (q, k, v):
        if t.shape == q.shape:
            with pytest.raises(ValueError):
                K().cross_fwd(q, k, v, 2, out=t)
    o, lse = K().cross_fwd(q, k, v, 2)
    for kw in (dict(dq=q), dict(dq=o), dict(dk=k), dict(dk=v), dict(dv=v)):
        with pytest.raises(ValueError):
            K().cross_bwd(q, k, v, o, lse, torch.zeros_like(q), 2, **kw)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Bc,Nq,Nk,H,G,hd,lens,mask,index", [
    (2, 2, 1, 700, 2, 2, 8, "empty", False, False),          # every lane layout: 1 to 32 lanes per row
    (3, 3, 1, 700, 4, 2, 16, "ragged", True, False),
    (3, 3, 5, 333, 3, 1, 24, "ragged", False, False),        # 15 rows
    (2, 2, 4, 517, 4, 1, 40, None, True, False),             # 16 rows, the whole list at once
    (4, 4, 2, 129, 2, 1, 64, "ragged", False, False),        # one state in the last tile
    (2, 2, 1, 1300, 2, 1, 96, "empty", True, False),
    (2, 2, 3, 401, 3, 3, 128, None, False, False),
    (7, 1, 1, 150, 4, 2, 32, None, True, False),             # one context for all
    (23, 8, 1, 260, 2, 1, 80, "ragged", True, True),         # a list of more than 16 rows for one, of none for others
    (70, 12, 1, 64, 2, 2, 64, "empty", False, True),         # an index longer than a wave
    (4, 1, 1, 150, 2, 2, 104, None, True, False),
])
def test_cross_short_row_lists(B, Bc, Nq, Nk, H, G, hd, lens, mask, index, dtype):
    kn = K()
    q, k, v, d_o, L, M, I = inputs(dtype, B, Bc, Nq, Nk, H, G, hd, lens, mask, index, seed=Nk + hd)
    if index:
        I[1], I[B - 1] = -3, Bc                               # no context: no gradient, zeros in dq
        I[2:14] = 3
    val, tol = reference(q, k, v, H, G, L, M, I, d_o=d_o)
    kp, vp = poison(k, v, L, M)
    dq_, dk_, dv_, do_, dL, dM, dI = cuda(q, kp, vp, d_o, L, M, I)
    kw = dict(kv_heads=G, lens=dL, mask=dM, index=dI)
    o, lse = kn.cross_fwd(dq_, dk_, dv_, H, **kw)
    first = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    rows = B * Nq * H // G / Bc                               # (up to 6 rows per context on average in bf16, 16 in fp32)
    assert kn.last_variant().startswith("cross_bwd_one") == (rows <= (6 if dtype == BF16 else 16))
    for name, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *first)):
        check(name, t, val, tol)
    again = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,Bc,Nq,Nk,H,G,hd,lens,mask,index,p", [
    (2, 2, 17, 300, 2, 2, 8, "ragged", False, False, 0.0),           # every width; 17 rows: one tile, half of it empty
    (3, 3, 32, 129, 2, 2, 24, "empty", True, False, 0.0),            # a whole tile; one state in the last workgroup
    (2, 2, 3, 700, 7, 1, 64, "ragged", True, False, 0.0),            # seven heads of a group
    (2, 2, 5, 260, 8, 2, 80, "ragged", False, False, 0.0),
    (1, 1, 30, 100, 1, 1, 128, None, True, False, 0.0),              # one workgroup: no partials
    (9, 1, 3, 200, 2, 2, 32, None, True, False, 0.0),                # one context for all: rows of nine samples in a tile
    (23, 4, 5, 333, 2, 2, 40, "ragged", True, True, 0.0),            # lists of several tiles, and empty ones
    (70, 9, 3, 150, 2, 2, 64, "empty", False, True, 0.0),
    (2, 2, 20, 140, 4, 4, 104, "ragged", False, False, 0.25),        # dropout
])
def test_cross_middle_row_lists(B, Bc, Nq, Nk, H, G, hd, lens, mask, index, p, dtype):
    kn = K()
    q, k, v, d_o, L, M, I = inputs(dtype, B, Bc, Nq, Nk, H, G, hd, lens, mask, index, seed=Nk + hd)
    if index:
        I[1], I[B - 1] = -3, Bc                               # no context: no gradient, zeros in dq
        I[2:14] = 3
    keep = None
    if p:                                                     # the mask, read off with unit values, a head width at a time
        cols = []
        for k0 in range(0, Nk, hd):
            eye = torch.zeros(Bc, Nk, G, hd)
            n = min(hd, Nk - k0)
            eye[:, torch.arange(k0, k0 + n), :, torch.arange(n)] = 1.0
            z, _ = kn.cross_fwd(q.cuda(), k.cuda(), eye.reshape(Bc, Nk, -1).to(dtype).cuda(), H, drop_p=p, drop_seed=5)
            cols.append((z.float().cpu().reshape(B, Nq, H, hd).permute(0, 2, 1, 3)[..., :n] > 0).double())
        keep = torch.cat(cols, -1) / (1.0 - round(p * 32768) / 32768)
    val, tol = reference(q, k, v, H, G, L, M, I, d_o=d_o, keep=keep)
    kp, vp = poison(k, v, L, M)
    dq_, dk_, dv_, do_, dL, dM, dI = cuda(q, kp, vp, d_o, L, M, I)
    kw = dict(kv_heads=G, lens=dL, mask=dM, index=dI, drop_p=p, drop_seed=5)
    o, lse = kn.cross_fwd(dq_, dk_, dv_, H, **kw)
    first = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    assert kn.last_variant().startswith("cross_bwd_rows") or (dtype == F32 and B * Nq * H // G <= 16 * Bc)
    for name, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *first)):
        check(name, t, val, tol)
    again = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,Nk,variant", [(1, 150, "cross_bwd_one"), (25, 150, "cross_bwd_rows"), (200, 150, "cross_bwd<"), (200, 20, "cross_bwd_few")])
def test_cross_table_of_more_contexts_than_samples(Nq, Nk, variant, dtype):
    """The form goes by the contexts that can have samples; the others get zeros."""
    kn = K()
    B, Bc, H, hd = 2, 50, 2, 64
    q, k, v, d_o, L, M, I = inputs(dtype, B, Bc, Nq, Nk, H, H, hd, "ragged", True, True, seed=Nq + Nk)
    I[:] = torch.tensor([7, 30])
    L[7], L[30] = Nk, Nk // 2
    val, tol = reference(q, k, v, H, H, L, M, I, d_o=d_o)
    dq_, dk_, dv_, do_, dL, dM, dI = cuda(q, *poison(k, v, L, M), d_o, L, M, I)
    kw = dict(lens=dL, mask=dM, index=dI)
    o, lse = kn.cross_fwd(dq_, dk_, dv_, H, **kw)
    grads = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, H, **kw)
    assert kn.last_variant().startswith(variant)
    for name, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *grads)):
        check(name, t, val, tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cross_single_query_long_stream_keeps_its_weights(dtype):
    """512 workgroups, so each streams its 4096 states alone, with scores around 369, whose product with log2(e) is rounded by
    2.9e-5: were that left in the factor of a step, it would grow with every step.  The scores 41 * 9 - j are exact in both types.
    Errors: lse rounds log2(e) and ln(2), their products and the last sum (4 u |lse|), the logarithm of at most 2^12 by 2 ulp
    (17 u); a weight is off by the argument of its exponential (at most 8.7 + 2.9e-5 / u, rounded: 9 u), the exponential (2 u),
    the adds of its lane (4 states a step, 4 waves, 64 / lanes-per-state states each) and 12 more in the joins."""
    kn = K()
    B, Nk, hd = 512, 4096, 128
    j = torch.randint(0, 7, (Nk,), generator=torch.Generator().manual_seed(1)).double()
    j[:64] = 0
    q, k, v = torch.zeros(B, 1, hd), torch.zeros(1, Nk, hd), torch.zeros(1, Nk, hd)
    q[..., 0], q[..., 1] = 41.0, 1.0
    k[0, :, 0], k[0, :, 1] = 9.0, -j.float()
    v[0, Nk // 2:] = 1.0
    o, lse = kn.cross_fwd(*(t.to(dtype).cuda() for t in (q, k, v)), 1, scale=1.0)
    assert kn.last_variant().startswith("cross_one")
    w = torch.exp(-j)
    want_lse, want_o = 369 + math.log(float(w.sum())), float(w[Nk // 2:].sum() / w.sum())
    rel = (9 + 2 + Nk // (4 * (64 // (16 if dtype == BF16 else 32))) + 12) * U
    assert float((lse.double().cpu() - want_lse).abs().max()) <= 4 * U * want_lse + 17 * U + rel
    assert float((o.double().cpu()[..., 0] - want_o).abs().max()) <= (2 * rel + 2 * U + (2.0 ** -8 if dtype == BF16 else U)) * want_o


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,Nk,hd", [(40, 20, 32), (40, 40, 32), (300, 13, 32), (300, 30, 32), (300, 40, 32), (300, 77, 16), (300, 90, 16), (200, 300, 64), (200, 900, 128),
                                      (20, 300, 64), (1, 300, 64), (4, 50, 32)])
@pytest.mark.parametrize("kind", ["lens", "mask"])
def test_cross_no_valid_state_whatever_the_query_holds(kind, Nq, Nk, hd, dtype):
    """Samples without a valid state get o = 0, lse = -infinity and no gradient also under NaN and infinite queries and output
    gradients, in every form."""
    kn = K()
    q, k, v, d_o, *_ = inputs(dtype, 3, 3, Nq, Nk, 2, 2, hd, None, False, False, seed=Nq + Nk)
    q[0], q[1], d_o[0] = float("nan"), float("inf"), float("nan")
    lens = torch.tensor([0, 0, Nk], dtype=torch.int32) if kind == "lens" else None
    mask = torch.tensor([[False], [False], [True]]).expand(3, Nk).contiguous() if kind == "mask" else None
    q, k, v, d_o, lens, mask = cuda(q, k, v, d_o, lens, mask)
    o, lse = kn.cross_fwd(q, k, v, 2, lens=lens, mask=mask)
    assert bool((o[:2] == 0).all()) and bool((lse[:2] == -math.inf).all()) and bool(torch.isfinite(lse[2]).all())
    for t in kn.cross_bwd(q, k, v, o, lse, d_o, 2, lens=lens, mask=mask):
        assert bool((t[:2] == 0).all()) and bool(torch.isfinite(t[2]).all())


def test_cross_refuses_outputs_that_share_memory():
    """With one another (the same tensor for two gradients, views that overlap) or with an operand, from another start; slices
    of one fused buffer are fine."""
    kn = K()
    buf = torch.zeros(2, 7, 96, dtype=BF16, device="cuda")
    q, k, v = (torch.randn(2, 7, 32, device="cuda").to(BF16) for _ in range(3))
    o, lse = kn.cross_fwd(q, k, v, 2)
    d_o, g = torch.randn_like(q), torch.zeros_like(q)
    for kw in (dict(dk=g, dv=g), dict(dq=g, dk=g), dict(dq=g, dv=g), dict(dk=buf[..., :32], dv=buf[..., 16:48]),
               dict(dq=buf[..., :32], dv=buf.view(-1)[8:8 + g.numel()].view_as(g))):
        with pytest.raises(ValueError):
            kn.cross_bwd(q, k, v, o, lse, d_o, 2, **kw)
    for out in (buf[..., 24:56], buf.view(-1)[8:8 + q.numel()].view_as(q)):
        with pytest.raises(ValueError):
            kn.cross_fwd(buf[..., :32], k, v, 2, out=out)
    want = kn.cross_bwd(q, k, v, o, lse, d_o, 2)
    kn.cross_bwd(q, k, v, o, lse, d_o, 2, dq=buf[..., :32], dk=buf[..., 32:64], dv=buf[..., 64:])
    assert all(torch.equal(a, b) for a, b in zip(want, buf.split(32, -1)))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,Nk", [(130, 130), (130, 70), (20, 130), (1, 130)])
def test_cross_rows_far_apart(Nq, Nk, dtype):
    """Rows so far apart (24 MiB in bf16, 40 MiB in fp32; 64 MiB is the limit) that 32 bits do not hold a step of the staging
    loads, which then go by plain addresses: queries, states, gradients and results, with masked states."""
    kn = K()
    ld = (24 << 20) // 2 if dtype == BF16 else (40 << 20) // 4
    base = torch.empty(1, max(Nq, Nk), ld, dtype=dtype, device="cuda")      # 3.0 and 5.1 GiB
    q, k, v, d_o, _, M, _ = inputs(dtype, 1, 1, Nq, Nk, 1, 1, 16, None, True, False, seed=Nq + Nk)
    val, tol = reference(q, k, v, 1, 1, None, M, d_o=d_o)
    at = {}
    for i, (name, t) in enumerate((("q", q), ("k", k), ("v", v), ("d_o", d_o), ("o", q), ("dq", q), ("dk", k), ("dv", k))):
        at[name] = base[:, :t.shape[1], 64 * i:64 * i + 16]
        at[name].copy_(t)
    o, lse = kn.cross_fwd(at["q"], at["k"], at["v"], 1, mask=M.cuda(), out=at["o"])
    grads = kn.cross_bwd(at["q"], at["k"], at["v"], o, lse, at["d_o"], 1, mask=M.cuda(), dq=at["dq"], dk=at["dk"], dv=at["dv"])
    for name, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *grads)):
        check(name, t, val, tol)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Nq,Nk,hd,variant", [(1, 300, 64, "cross_bwd_one"), (20, 150, 64, "cross_bwd_rows"), (70, 150, 64, "cross_bwd<"),
                                              (70, 40, 32, "cross_bwd_few")])
def test_cross_half_of_the_samples_on_one_context(Nq, Nk, hd, variant, dtype):
    """The form goes by the average list; one list of 33 samples among lists of one or none."""
    kn = K()
    B = 66
    q, k, v, d_o, L, _, I = inputs(dtype, B, B, Nq, Nk, 1, 1, hd, "ragged", False, True, seed=Nq)
    I[:] = torch.arange(B, dtype=torch.int32)
    I[::2] = 5
    L[5] = Nk
    val, tol = reference(q, k, v, 1, 1, L, None, I, d_o=d_o)
    dq_, dk_, dv_, do_, dL, dI = cuda(q, *poison(k, v, L, None), d_o, L, I)
    o, lse = kn.cross_fwd(dq_, dk_, dv_, 1, lens=dL, index=dI)
    grads = kn.cross_bwd(dq_, dk_, dv_, o, lse, do_, 1, lens=dL, index=dI)
    assert kn.last_variant().startswith(variant)
    for name, t in zip(("o", "lse", "dq", "dk", "dv"), (o, lse, *grads)):
        check(name, t, val, tol)
