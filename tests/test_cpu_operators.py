"""CPU: what the rotary and cross-attention front-ends refuse, and that the C entries refuse it too (no launch is made: every
case here is turned away before one)."""
import ctypes

import pytest
import torch

from diffusion_model_amd import _lib
from diffusion_model_amd import kernels as K

BF16, F32 = torch.bfloat16, torch.float32


def plan(hd=32, axes=(16, 16), **kw):
    return K.rope_plan(hd, axes, device="cpu", **kw)


@pytest.mark.parametrize("hd,axes,kw", [
    (32, (), {}), (32, (8, 8, 8, 8), {}), (32, (15,), {}), (32, (0, 16), {}), (32, (32, 2), {}), (33, (16,), {}),
    (2050, (16,), {}), (32, (16,), dict(pairing="other")), (32, (16,), dict(theta=0.0)), (32, (16,), dict(theta=float("inf")))])
def test_rope_plan_refusals(hd, axes, kw):
    with pytest.raises(ValueError):
        plan(hd, axes, **kw)


def test_rope_plan_values():
    import math
    p = plan(40, (4, 6), theta=100.0)
    want = [100.0 ** (-2 * i / d) / (2 * math.pi) for d in (4, 6) for i in range(d // 2)]
    assert p.freq.tolist() == want and p.axis.tolist() == [0, 0, 1, 1, 1] and p.rot == 10


X = torch.zeros(2, 6, 64)


@pytest.mark.parametrize("x,heads,kw", [
    (X[0], 2, dict(grid=(2, 3))), (X.half(), 2, dict(grid=(2, 3))), (X, 3, dict(grid=(2, 3))), (X, 0, dict(grid=(2, 3))),
    (X, 2, {}), (X, 2, dict(grid=(2, 3), positions=torch.zeros(6, 2))), (X, 2, dict(grid=(2, 4))), (X, 2, dict(grid=(6,))),
    (X, 2, dict(grid=(-2, -3))), (X, 2, dict(positions=torch.zeros(6, 3))), (X, 2, dict(positions=torch.zeros(3, 6, 2))),
    (X, 2, dict(positions=torch.zeros(6, 2, dtype=torch.int64))), (X, 2, dict(positions=torch.zeros(2, 6).T)),
    (X, 2, dict(grid=(2, 3), out=torch.zeros(2, 6, 32))), (X, 2, dict(grid=(2, 3), out=X.to(BF16))),
    (torch.zeros(1, 1, 65536), 2048, dict(grid=(1, 1))),
    (X, 2, dict(grid=(2, 3)))])                       # the last one: everything fits, but no tensor is on the GPU
def test_rope_refusals(x, heads, kw):
    with pytest.raises(ValueError):
        K.rope(x, heads, plan(), **kw)


Q, KV = torch.zeros(2, 5, 64), torch.zeros(2, 7, 64)


@pytest.mark.parametrize("q,k,v,heads,kw", [
    (Q[0], KV, KV, 2, {}), (Q, KV[0], KV[0], 2, {}), (Q.half(), KV.half(), KV.half(), 2, {}), (Q.to(BF16), KV, KV, 2, {}),
    (Q, KV, KV[:, :5], 2, {}), (Q, KV, KV.to(BF16), 2, {}), (Q, KV, KV, 3, {}), (Q, KV, KV, 0, {}), (Q, KV, KV, 2, dict(kv_heads=1)),
    (Q, KV, KV, 4, dict(kv_heads=3)), (Q, KV, KV, 2, dict(kv_heads=0)),
    (Q, KV, KV, 16, {}),                                                               # head width 4
    (torch.zeros(2, 5, 272), torch.zeros(2, 7, 272), torch.zeros(2, 7, 272), 2, {}),   # head width 136
    (torch.zeros(4, 5, 64), KV, KV, 2, {}),                                            # 2 contexts for 4 samples
    (Q, KV[:0], KV[:0], 2, dict(index=torch.zeros(2, dtype=torch.int32))),
    (Q, KV, KV, 2, dict(lens=torch.zeros(2))), (Q, KV, KV, 2, dict(lens=torch.zeros(3, dtype=torch.int32))),
    (Q, KV, KV, 2, dict(index=torch.zeros(2, dtype=torch.int64))), (Q, KV, KV, 2, dict(index=torch.zeros(1, dtype=torch.int32))),
    (Q, KV, KV, 2, dict(mask=torch.zeros(2, 7))), (Q, KV, KV, 2, dict(mask=torch.zeros(7, 2, dtype=torch.bool).T)),
    (Q, KV, KV, 2, dict(mask=torch.zeros(2, 1, 7, dtype=torch.bool))),
    (Q, KV, KV, 2, dict(scale=0.0)), (Q, KV, KV, 2, dict(scale=-1.0)), (Q, KV, KV, 2, dict(scale=float("nan"))),
    (Q, KV, KV, 2, dict(drop_p=1.0)), (Q, KV, KV, 2, dict(drop_p=-0.1)),
    (Q, KV, KV, 2, {})])                              # the last one: everything fits, but no tensor is on the GPU
def test_cross_refusals(q, k, v, heads, kw):
    with pytest.raises(ValueError):
        K.cross_fwd(q, k, v, heads, **kw)
    with pytest.raises(ValueError):
        K.cross_bwd(q, k, v, q, torch.zeros(q.shape[0], max(heads, 1), q.shape[1] if q.dim() > 2 else 1), q, heads, **kw)


def cross_struct(**kw):
    """Arguments that a launch would take, with addresses that are never read (every test changes one to be refused)."""
    a = _lib.CrossArgs()
    for n in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "workspace"):
        setattr(a, n, 4096)
    for n in ("ldq", "ldk", "ldv", "ldo", "lddo", "lddq", "lddk", "lddv"):
        setattr(a, n, 64)
    a.B = a.Bc = 2
    a.heads = a.kv_heads = 2
    a.Nq, a.Nk, a.hd, a.dtype, a.scale, a.ws_bytes = 5, 7, 32, 0, 0.2, 1 << 30
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(B=0), dict(Bc=0), dict(Bc=1, B=2, index=None, k=None), dict(B=3), dict(heads=3), dict(kv_heads=0), dict(Nq=0), dict(Nk=-1),
    dict(hd=4), dict(hd=36), dict(hd=136), dict(dtype=2), dict(scale=0.0), dict(scale=float("nan")), dict(drop_p=1.0),
    dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(lse=None), dict(q=4098), dict(ldq=63), dict(ldq=32), dict(ldk=60)])
def test_cross_entry_points_refuse(kw):
    L = _lib.lib()
    a = cross_struct(**kw)
    assert L.dm_cross_fwd(ctypes.byref(a), None) == -1
    assert L.dm_cross_bwd(ctypes.byref(a), None) == -1


@pytest.mark.parametrize("kw", [dict(d_o=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(lddq=60), dict(workspace=None),
                                dict(ws_bytes=4), dict(workspace=4100)])
def test_cross_backward_entry_point_refuses(kw):
    assert _lib.lib().dm_cross_bwd(ctypes.byref(cross_struct(Nk=600, **kw)), None) == -1      # (so many keys need scratch)


def test_cross_workspace_bytes():
    L = _lib.lib()
    assert L.dm_cross_fwd_workspace_bytes(ctypes.byref(cross_struct())) == 0
    assert L.dm_cross_fwd_workspace_bytes(ctypes.byref(cross_struct(Nq=1, Nk=4096))) > 0     # few rows: keys are split
    assert L.dm_cross_bwd_workspace_bytes(ctypes.byref(cross_struct(Nk=600))) >= 2 * 2 * 5 * 4
    shared = cross_struct(B=3, Bc=1, Nq=9)                                     # few keys, one context for all: a partial per sample
    assert L.dm_cross_bwd_workspace_bytes(ctypes.byref(shared)) == 3 * 2 * 2 * 7 * 32 * 4
    one = cross_struct(B=3, Bc=1, Nq=2, Nk=300)                                      # few rows: a partial of dQ per 128 states
    assert L.dm_cross_bwd_workspace_bytes(ctypes.byref(one)) == 3 * 3 * 2 * 2 * 32 * 4
    assert L.dm_cross_bwd_workspace_bytes(ctypes.byref(cross_struct(B=3, Bc=1, Nq=2))) == 0
    shared.workspace = None
    assert L.dm_cross_bwd(ctypes.byref(shared), None) == -1
    assert L.dm_cross_fwd_workspace_bytes(None) == 0 and L.dm_cross_fwd(None, None) == -1 and L.dm_cross_bwd(None, None) == -1
    crowd = cross_struct(B=4096, Bc=1, Nq=64, Nk=16384)                        # the partial results of key splits stay below 1 GiB
    assert L.dm_cross_fwd_workspace_bytes(ctypes.byref(crowd)) < 1 << 30
    # contexts that no sample uses leave the way the work is done as it is: long rows keep the kernels of long rows
    own, table = (cross_struct(B=2, Bc=n, Nq=2304, Nk=77, index=4096) for n in (2, 1000))
    assert L.dm_cross_bwd_workspace_bytes(ctypes.byref(table)) == L.dm_cross_bwd_workspace_bytes(ctypes.byref(own))
    table.Nk = 600
    assert L.dm_cross_bwd_workspace_bytes(ctypes.byref(table)) < 1 << 29
    few = cross_struct(Nq=1, Nk=4096, workspace=None)
    assert L.dm_cross_fwd(ctypes.byref(few), None) == -1


def rope_struct(**kw):
    a = _lib.RopeArgs()
    a.x = a.y = a.freq = a.axis = 4096
    a.ldx = a.ldy = 64
    a.B, a.N, a.heads, a.hd, a.rot, a.axes = 2, 6, 2, 32, 32, 2
    a.grid[0], a.grid[1] = 2, 3
    for n, v in kw.items():
        if n == "grid":
            for i, g in enumerate(v):
                a.grid[i] = g
        else:
            setattr(a, n, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(y=None), dict(freq=None), dict(axis=None), dict(B=0), dict(N=0), dict(heads=0), dict(hd=0), dict(hd=31),
    dict(rot=0), dict(rot=34), dict(rot=15), dict(axes=0), dict(axes=4), dict(dtype=2), dict(pairing=2), dict(ldx=32), dict(ldy=63),
    dict(grid=(2, 4)), dict(grid=(0, 3)), dict(grid=(-2, -3)), dict(grid=(1 << 30, 1 << 30)), dict(heads=2048)])
def test_rope_entry_point_refuses(kw):
    assert _lib.lib().dm_rope(ctypes.byref(rope_struct(**kw)), None) == -1


C3 = torch.zeros(2, 7, 48)


@pytest.mark.parametrize("x,kw", [
    (C3[0], {}), (C3, dict(lens=torch.zeros(3, dtype=torch.int32))), (C3, dict(lens=torch.zeros(2, dtype=torch.int64))),
    (C3, dict(mask=torch.zeros(2, 6, dtype=torch.bool))), (C3, dict(index=torch.zeros(5, dtype=torch.int32))),
    (C3, {})])                                        # the last one: everything fits, but no tensor is on the GPU
def test_context_rows_refusals(x, kw):
    with pytest.raises(ValueError):
        K.context_rows(x, 4, **kw)


def test_context_rows_entry_point_refuses():
    f = _lib.lib().dm_context_rows
    for args in ((None, 4096, 0, 2, 7, 48, None, None, None, 2), (4096, None, 0, 2, 7, 48, None, None, None, 2),
                 (4096, 4096, 0, 0, 7, 48, None, None, None, 2), (4096, 4096, 0, 2, 0, 48, None, None, None, 2),
                 (4096, 4096, 0, 2, 7, 0, None, None, None, 2), (4096, 4096, 0, 2, 7, 48, None, None, 4096, 0)):
        assert f(*args, None) == -1
    assert f(4096, 4096, 0, 1 << 20, 1 << 10, 48, None, None, None, 2, None) == -3       # more rows than a launch holds


@pytest.mark.parametrize("kw", [dict(B=3, Bc=3, Nq=2, Nk=20), dict(B=4, Bc=4, Nq=20, Nk=150, hd=128, ldq=256, ldk=256, ldv=256),
                                dict(B=2, Bc=2, Nq=64, Nk=20), dict(B=2, Bc=2, Nq=200, Nk=400)])
def test_cross_workspace_bytes_read_the_fields_that_the_header_names(kw):
    """Scratch sized from the named fields alone is the scratch that the call asks for; whether index is NULL is one of them."""
    import os
    L = _lib.lib()
    names = ("B", "Bc", "heads", "kv_heads", "Nq", "Nk", "hd", "dtype", "index")
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "dm_hip.h")).read()
    said = header[header.index("/* Scratch for these sizes"):header.index("long dm_cross_fwd_workspace_bytes")]
    assert all(n in said for n in names)
    sizes = []
    for index in (None, 4096):
        full, bare = cross_struct(**kw, index=index, lens=4096, mask=4096), _lib.CrossArgs()
        for n in names:
            setattr(bare, n, getattr(full, n))
        for f in (L.dm_cross_fwd_workspace_bytes, L.dm_cross_bwd_workspace_bytes):
            assert f(ctypes.byref(bare)) == f(ctypes.byref(full))
        sizes.append(L.dm_cross_bwd_workspace_bytes(ctypes.byref(bare)))
    if kw["Nk"] < 200:
        assert sizes[0] != sizes[1]


def test_partial_sampling_makes_its_contexts_once_per_joining_group(monkeypatch):
    """sample_from: the table goes to the device, is gathered and its ids are looked over when samples join the walk, not in
    every step."""
    from diffusion_model_amd.sampler import CFGSampler
    from diffusion_model_amd.utils import DDPM_beta_t_cosine_scheduler
    seen, made = [], []

    class Model:
        def eval(self):
            return self

        def _fwd(self, zz, tt, ctx, cmap=None):
            n = zz.shape[0]
            index = torch.arange(ctx.shape[0]) if cmap is None or cmap.index is None else cmap.index.long()
            seen.append((int(tt[0]), ctx[index][:, 0, 0].tolist(), None if cmap is None else cmap.lens.tolist()))
            assert index.numel() == n
            return torch.zeros_like(zz), None

    monkeypatch.setattr(K, "cfg_ddpm_step", lambda z, v_u, v_c, noise, coef: z)
    make = CFGSampler._contexts
    monkeypatch.setattr(CFGSampler, "_contexts", lambda self, ids: made.append(ids.tolist()) or make(self, ids))
    table = torch.arange(4.0)[:, None, None].expand(4, 7, 8).contiguous()
    labels, starts = torch.tensor([0, 1, 2, 1, 3]), [0, 6, 9, 6, 9]
    for lens in (None, torch.tensor([7, 3, 5, 1])):
        seen.clear(), made.clear()
        CFGSampler(Model(), DDPM_beta_t_cosine_scheduler(50), table, 3, context_lens=lens).sample_from(torch.zeros(5, 1, 2, 2), labels, starts)
        assert made == [[3, 3, 2, 3], [3] * 4 + [2, 3, 1, 1], [3] * 5 + [2, 3, 1, 1, 0]]
        assert [t for t, *_ in seen] == list(range(9, -1, -1))
        for t, ids, _ in seen:
            assert ids == made[0 if t > 6 else (1 if t > 0 else 2)]


def test_shared_memory_of_row_views():
    """_share against the sets of addresses, for views of one buffer with the rows that the front-ends take."""
    import random
    rng, buf, both = random.Random(3), torch.zeros(400), [0, 0]

    def view():
        while True:
            n0, n1, w, at = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 8), rng.randint(0, 200)
            ld = rng.choice([16, 16, 16, w, 11])
            if w <= ld and at + (n0 * n1 - 1) * ld + w <= 400:
                return buf.as_strided((n0, n1, w), (n1 * ld, ld, 1), at)

    def cells(t):
        return {t.storage_offset() + i * t.stride(0) + j * t.stride(1) + c for i in range(t.shape[0]) for j in range(t.shape[1]) for c in range(t.shape[2])}

    for _ in range(4000):
        a, b = view(), view()
        share = bool(cells(a) & cells(b))
        (_, la, n, _), (_, lb, m, _) = K._span(a), K._span(b)
        if n == 1 or m == 1 or la == lb:
            assert K._share(a, b) == share == K._share(b, a)
            both[share] += 1
        elif share:
            assert K._share(a, b) and K._share(b, a)
    assert min(both) > 300
    assert not K._share(buf[:0].view(1, 0, 4), buf.view(1, 100, 4)) and K._share(buf[:1].expand(2, 3, 1), buf.view(1, 100, 4))


def test_rope_entry_point_refuses_other_rows_at_the_same_start():
    assert _lib.lib().dm_rope(ctypes.byref(rope_struct(ldx=192)), None) == -1


@pytest.mark.parametrize("kw", [dict(mask=torch.zeros(2, 7)), dict(mask=[[0.0, float("-inf")]]), dict(lens=torch.tensor([1.0, 2.0])),
                                dict(lens=[True, False]), dict(index=torch.tensor([0.0])), dict(index=torch.zeros(2, dtype=torch.bool))])
def test_context_map_refuses_other_kinds_of_numbers(kw):
    from diffusion_model_amd.unet import ContextMap
    with pytest.raises(ValueError):
        ContextMap.of("cpu", **kw)


def test_context_map_types():
    from diffusion_model_amd.unet import ContextMap
    m = ContextMap.of("cpu", [3, 0], torch.tensor([[1, 0], [0, 2]]), torch.tensor([1, 0, 1]))
    assert (m.lens.dtype, m.mask.dtype, m.index.dtype) == (torch.int32, torch.bool, torch.int32)
    assert m.mask.tolist() == [[True, False], [False, True]] and ContextMap.of("cpu") is None
    assert ContextMap.of("cpu", lens=[]).lens.shape == (0,)


@pytest.mark.parametrize("kw", [dict(Nq=1), dict(Nq=1, Nk=600), dict(Nq=5), dict(Nq=20, Nk=600), dict(Nq=40, Nk=600, ldq=128),
                                dict(Nq=40, Nk=20), dict(Nq=200, Nk=600, Bc=1)])
def test_cross_grids_that_hip_does_not_take(kw):
    """A launch holds fewer than 2^32 threads along its grid: more samples and heads than 2^24 workgroups of 256 are refused."""
    L = _lib.lib()
    a = cross_struct(**{**dict(B=1 << 23, Bc=1 << 23, ws_bytes=1 << 62), **kw})
    assert L.dm_cross_fwd(ctypes.byref(a), None) == -3
    assert L.dm_cross_bwd(ctypes.byref(a), None) == -3


def test_rope_grids_that_hip_does_not_take():
    a = rope_struct(B=1 << 20, N=1 << 10, heads=32, ldx=1024, ldy=1024, axes=1, grid=(1 << 10, 0))
    assert _lib.lib().dm_rope(ctypes.byref(a), None) == -3
