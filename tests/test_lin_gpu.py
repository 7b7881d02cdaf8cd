"""Linear attention with a decay per head on the GPU, against its definition in
64 bits.

Tolerances, from the arithmetic (u = half a step of the I/O type, w = 2^-8 of
bf16, e = 2^-24 of fp32; `abs` the sum of the terms' absolute values):

* decode keeps everything in fp32: a state element has the gate's exp (a few
  units, growing with |g| through the product with log2 e) and two roundings; an
  output adds the d_k products and one rounding to the I/O type.
* prefill rounds the decayed scores to the I/O type (u), the scaled queries and
  the states they meet to bf16 (2 w), and the output (u).  The states' updates
  split the decayed values into two parts of the I/O type: what is left is
  u^2 of each term, and in f16 half a step of its smallest number.
"""
from __future__ import annotations

import pytest
import torch

from conftest import graft
from lin_oracle import half_step, steps

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -24
W = half_step(torch.bfloat16)


def make(lead, Hqk, Hv, dk, dv, io, seed, gmin=-0.2, g_dtype=torch.float32, gate="token"):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(*lead, Hqk, dk, generator=gen).to(io)
    k = torch.randn(*lead, Hqk, dk, generator=gen).to(io)
    v = torch.randn(*lead, Hv, dv, generator=gen).to(io)
    g = (torch.rand(*(lead if gate == "token" else ()), Hv, generator=gen) * gmin).to(g_dtype)
    return q, k, v, g


def check_prefill(o, S, ref, io, k, v):
    ro, rS, oa, Sa = ref
    u = half_step(io)
    tol = u * ro.abs() + (u + 2 * W + 64 * E) * oa + 1e-12
    assert bool(((o.double() - ro).abs() <= tol).all()), float(((o.double() - ro).abs() / tol).max())
    tiny = 2.0 ** -25 if io == torch.float16 else 0.0
    tolS = (u * u + 64 * E) * Sa + tiny * k.double().abs().sum(0).amax() + 1e-12
    assert bool(((S.double() - rS).abs() <= tolS).all()), float(((S.double() - rS).abs() / tolS).max())


# ------------------------------------------------------------------ decode


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 192), (128, 64), (128, 128), (256, 64), (256, 128)])
@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Hqk,Hv", [(1, 1, 1), (3, 2, 4), (37, 3, 3)])
def test_decode(pkg, dk, dv, io, B, Hqk, Hv):
    q, k, v, g = make((B,), Hqk, Hv, dk, dv, io, B + dk)
    S = torch.randn(B, Hv, dk, dv, generator=torch.Generator().manual_seed(1))
    st = S.to(DEV)
    o = pkg.lin_decode(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), st, scale=0.5, check=True).cpu()
    check_decode(o, st.cpu(), q, k, v, g, S, 0.5, io)


def check_decode(o, st, q, k, v, g, S, scale, io, rows=None):
    dk = q.shape[-1]
    for b in rows if rows is not None else range(q.shape[0]):
        gb = g[b : b + 1] if g.dim() == 2 else g[None]
        ro, rS, oa, Sa = steps(q[b : b + 1], k[b : b + 1], v[b : b + 1], gb, S[b], scale)
        c = 8 + 4 * float(gb.float().abs().max())
        assert bool(((st[b].double() - rS).abs() <= c * E * Sa).all())
        tol = half_step(io) * ro[0].abs() + (dk + c) * E * oa[0] + 2.0 ** -25 * (io == torch.float16)
        assert bool(((o[b].double() - ro[0]).abs() <= tol).all())


@pytest.mark.parametrize("gate", ["token", "head"])
@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_decode_gates(pkg, gate, g_dtype):
    q, k, v, g = make((5,), 2, 2, 64, 64, torch.bfloat16, 3, gmin=-3.0, g_dtype=g_dtype, gate=gate)
    S = torch.randn(5, 2, 64, 64)
    st = S.to(DEV)
    args = [x.to(DEV) for x in (q, k, v, g)]
    o = pkg.lin_decode(*args, st, check=True).cpu()
    check_decode(o, st.cpu(), q, k, v, g, S, 1.0, torch.bfloat16)
    lin = S.to(DEV)
    o2 = pkg.lin_decode(*args[:3], args[3].float().exp(), lin, gate="linear", check=True).cpu()
    torch.testing.assert_close(lin.cpu(), st.cpu(), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(o2, o, rtol=2 * half_step(torch.bfloat16), atol=1e-3)


def test_decode_reset_gate_forgets(pkg):
    """g = -inf (decay 0) drops the old state whole."""
    q, k, v, _ = make((2,), 1, 2, 64, 64, torch.bfloat16, 4)
    g = torch.tensor([[float("-inf"), 0.0], [0.0, float("-inf")]])
    S = torch.randn(2, 2, 64, 64)
    st = S.to(DEV)
    o = pkg.lin_decode(q.to(DEV), k.to(DEV), v.to(DEV), g.to(DEV), st, check=True).cpu()
    kv = k.double()[:, :, :, None] * v.double()[:, :, None, :]
    want = torch.where(g[:, :, None, None] < 0, 0.0, S.double()) + kv
    assert float((st.cpu().double() - want).abs().max()) <= 4 * E * float(want.abs().max())
    assert torch.isfinite(o).all()


def test_decode_pages_idle_bad_and_shared_rows(pkg):
    B, P = 9, 12
    q, k, v, g = make((B,), 2, 4, 64, 128, torch.float16, 5)
    pool = torch.randn(P, 4, 64, 128)
    index = torch.tensor([3, -1, 0, 11, 3, 12, 7, -5, 2 ** 31 - 1], dtype=torch.int32)
    good = {0: 3, 2: 0, 3: 11, 6: 7}  # row 4 wants the page of row 0; 5 and 8 lie outside
    st = pool.to(DEV)
    out = torch.full((B, 4, 128), float("nan"), dtype=torch.float16, device=DEV)
    args = [x.to(DEV) for x in (q, k, v, g)]
    with pytest.raises(pkg.GDNError, match="index"):
        pkg.lin_decode(*args, st, index=index.to(DEV), out=out, check=True)
    o, st = out.cpu(), st.cpu()
    rows = sorted(good)
    check_decode(o[rows], st[[good[r] for r in rows]], q[rows], k[rows], v[rows], g[rows],
                 pool[[good[r] for r in rows]], 1.0, torch.float16)
    idle = [r for r in range(B) if r not in good]
    assert bool((o[idle] == 0).all())
    rest = [p for p in range(P) if p not in good.values()]
    assert torch.equal(st[rest], pool[rest])
    pkg.check_device_status(torch.device(DEV))  # the report was cleared


def test_decode_strides_out_of_place_and_pool_slices(pkg):
    B, Hqk, Hv, d = 6, 2, 4, 64
    gen = torch.Generator().manual_seed(6)
    qkv = torch.randn(B, Hqk * 2 + Hv, d, generator=gen).to(torch.bfloat16).to(DEV)
    q, k, v = qkv[:, :Hqk], qkv[:, Hqk : 2 * Hqk], qkv[:, 2 * Hqk :]
    g = (-torch.rand(Hv, B, generator=gen)).to(DEV).t()
    layers = torch.randn(B, 3, Hv, d, d, generator=gen).to(DEV)
    new = torch.full((B, Hv, d, d), float("nan"), device=DEV)
    out = torch.zeros(B, 2, Hv, d, dtype=torch.bfloat16, device=DEV)
    before = layers.clone()
    pkg.lin_decode(q, k, v, g, layers[:, 1], out=out[:, 1], state_out=new, check=True)
    assert torch.equal(layers, before) and bool((out[:, 0] == 0).all())
    check_decode(out[:, 1].cpu(), new.cpu(), q.cpu(), k.cpu(), v.cpu(), g.cpu(), before[:, 1].cpu(), 1.0,
                 torch.bfloat16)


def test_decode_more_rows_than_a_grid_axis(pkg):
    B, d = 66000, 64
    q, k, v, g = make((B,), 1, 1, d, d, torch.bfloat16, 38)
    S = torch.randn(1, 1, d, d, generator=torch.Generator().manual_seed(39))
    st = S.to(DEV).repeat(B, 1, 1, 1)
    o = pkg.lin_decode(*(x.to(DEV) for x in (q, k, v, g)), st, check=True)
    rows = [0, 1, 65534, 65535, 65536, B - 1]
    check_decode(o[rows].cpu(), st[rows].cpu(), q[rows], k[rows], v[rows], g[rows], S.expand(len(rows), -1, -1, -1), 1.0,
                 torch.bfloat16)


def test_decode_large_pool_offsets(pkg):
    """Pages whose element offsets pass 32 bits."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    Hv, dk, dv = 32, 128, 128
    pool = torch.empty((1 << 32) // (Hv * dk * dv) + 3, Hv, dk, dv, device=DEV)
    P = pool.shape[0]
    pages = [P - 1, 0, P - 2]
    q, k, v, g = make((3,), 32, 32, dk, dv, torch.bfloat16, 7)
    S = torch.randn(3, Hv, dk, dv, generator=torch.Generator().manual_seed(8))
    pool[pages] = S.to(DEV)
    o = pkg.lin_decode(*(x.to(DEV) for x in (q, k, v, g)), pool,
                       index=torch.tensor(pages, dtype=torch.int32, device=DEV), check=True).cpu()
    check_decode(o, pool[pages].cpu(), q, k, v, g, S, 1.0, torch.bfloat16)


# ------------------------------------------------------------------ prefill


@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128)])
@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
def test_prefill(pkg, T, dk, dv, io):
    B, Hqk, Hv = 2, 1, 2
    q, k, v, g = make((B, T), Hqk, Hv, dk, dv, io, T + dk)
    S0 = torch.randn(B, Hv, dk, dv, generator=torch.Generator().manual_seed(T)) if T % 2 else None
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV) if S0 is not None else None,
                           scale=dk ** -0.5, check=True)
    for b in range(B):
        ref = steps(q[b], k[b], v[b], g[b], S0[b] if S0 is not None else torch.zeros(Hv, dk, dv), dk ** -0.5)
        check_prefill(o[b].cpu(), S[b].cpu(), ref, io, k[b], v[b])


@pytest.mark.parametrize("dv", [192, 256])
@pytest.mark.parametrize("B,Hqk,Hv", [(1, 1, 1), (1, 1, 5), (3, 2, 4)])
def test_prefill_wide_values_and_heads(pkg, dv, B, Hqk, Hv):
    T, dk, io = 150, 128, torch.bfloat16
    q, k, v, g = make((B, T), Hqk, Hv, dk, dv, io, dv)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), check=True)
    for b in range(B):
        ref = steps(q[b], k[b], v[b], g[b], torch.zeros(Hv, dk, dv), 1.0)
        check_prefill(o[b].cpu(), S[b].cpu(), ref, io, k[b], v[b])


@pytest.mark.parametrize("gate", ["token", "head"])
@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gmin", [0.0, -0.01, -5.0])
def test_prefill_gates(pkg, gate, g_dtype, gmin):
    T, d, io = 200, 64, torch.bfloat16
    q, k, v, g = make((1, T), 2, 2, d, d, io, 9, gmin=gmin, g_dtype=g_dtype, gate=gate)
    S0 = torch.randn(1, 2, d, d)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), check=True)
    gg = g[0] if gate == "token" else g.expand(T, 2)
    check_prefill(o[0].cpu(), S[0].cpu(), steps(q[0], k[0], v[0], gg, S0[0], 1.0), io, k[0], v[0])


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gmin,gmax", [(-1.0, 0.0), (-2.0, 0.0), (-2.5, 0.0), (-3.5, 0.0), (-0.4, 0.4), (0.0, 0.05)])
def test_prefill_gate_ranges(pkg, io, gmin, gmax):
    """Decays over a chunk from mild to beyond fp32's range, and gates that grow."""
    T, d = 300, 64
    q, k, v, _ = make((1, T), 1, 2, d, d, io, 18)
    g = gmin + (gmax - gmin) * torch.rand(1, T, 2, generator=torch.Generator().manual_seed(19))
    g[0, :, 1] = g[0, :, 1].sort().values  # and a head whose decay changes along the way
    S0 = torch.randn(1, 2, d, d)
    v = (v.float() * 2.0 ** -4).to(io)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=0.125, check=True)
    ro, rS, oa, Sa = steps(q[0], k[0], v[0], g[0], S0[0], 0.125)
    heads = [0, 1]
    if io == torch.float16 and gmax == 0.4:
        # the second head's exact outputs reach 2.3e13: no f16 holds them
        assert float(ro[:, 1].abs().max()) > torch.finfo(io).max
        heads = [0]
    check_prefill(o[0, :, heads].cpu(), S[0, heads].cpu(), (ro[:, heads], rS[heads], oa[:, heads], Sa[heads]), io,
                  k[0], v[0])


@pytest.mark.parametrize("gmin", [-0.5, -1.4, -2.5])
def test_prefill_large_values_under_strong_decay(pkg, gmin):
    """Sums that leave out the rows' factors stay within fp32's range, and rows of which the state
    before the chunk has all but vanished take at most 2^-80 of it (v is zero from token 120 on)."""
    T, d, io = 300, 64, torch.bfloat16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 44, gmin=gmin)
    v = (v.float() * 2.0 ** 36).to(io)
    v[:, 120:] = 0
    S0 = torch.randn(1, 2, d, d)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), check=True)
    ro, rS, oa, Sa = steps(q[0], k[0], v[0], g[0], S0[0], 1.0)
    for c in range(0, T, 128):
        at = steps(q[0, :c], k[0, :c], v[0, :c], g[0, :c], S0[0], 1.0)[3] if c else S0[0].double().abs()
        rows = slice(c, min(c + 128, T))
        oa[rows] += 2.0 ** -80 / (half_step(io) + 2 * W) * torch.einsum("td,hde->the", q[0, rows, 0].double().abs(), at)
    check_prefill(o[0].cpu(), S[0].cpu(), (ro, rS, oa, Sa), io, k[0], v[0])


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("g_reset", [float("-inf"), -200.0, -1e30])
def test_prefill_resets(pkg, g_reset, io):
    """A decay of zero at some tokens starts the sequence anew there, also inside a chunk."""
    T, d = 260, 64
    q, k, v, g = make((1, T), 1, 2, d, d, io, 10)
    g[0, [0, 5, 6, 127, 128, 200], 0] = g_reset
    g[0, :, 1] = g_reset
    S0 = torch.randn(1, 2, d, d)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), check=True)
    check_prefill(o[0].cpu(), S[0].cpu(), steps(q[0], k[0], v[0], g[0], S0[0], 1.0), io, k[0], v[0])


def test_prefill_packed_ragged_with_pages(pkg):
    Hqk, Hv, dk, dv, io = 1, 2, 128, 64, torch.float16
    lens = [5, 0, 130, 1, 128, 257, 0, 64]
    lead, tail = 3, 9  # rows before the first and behind the last sequence
    T = lead + sum(lens) + tail
    q, k, v, g = make((1, T), Hqk, Hv, dk, dv, io, 11)
    # nothing of the rows outside may reach a sequence
    for x in (q, k, v):
        x[0, :lead] = float("nan")
        x[0, T - tail :] = float("inf")
    cu = [lead]
    for n in lens:
        cu.append(cu[-1] + n)
    P = 11
    pool = torch.randn(P, Hv, dk, dv, generator=torch.Generator().manual_seed(12))
    index = torch.tensor([4, 9, 0, -1, 10, 2, -3, 7], dtype=torch.int32)
    st = pool.to(DEV)
    out = torch.full((1, T, Hv, dv), 7.0, dtype=io, device=DEV)
    o, fin = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), st, scale=0.1, out=out, index=index.to(DEV),
                             cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV), check=True)
    assert fin is st and o is out
    o, fin = o.cpu(), fin.cpu()
    assert bool((o[0, :lead] == 7).all()) and bool((o[0, T - tail :] == 7).all())
    kept = set(range(P))
    for n, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        p = int(index[n])
        S0 = pool[p] if p >= 0 else torch.zeros(Hv, dk, dv)
        ref = steps(q[0, a:b], k[0, a:b], v[0, a:b], g[0, a:b], S0, 0.1)
        if p >= 0:
            kept.discard(p)
            if b == a:
                assert torch.equal(fin[p], pool[p])
                continue
        elif b == a:
            continue
        check_prefill(o[0, a:b], fin[p] if p >= 0 else ref[1], ref, io, k[0, a:b], v[0, a:b])
    kept = sorted(kept)
    assert torch.equal(fin[kept], pool[kept])


def test_prefill_neighbours_of_other_sequences_stay_out(pkg):
    """A sequence that ends inside a chunk, next to one of NaN and infinities."""
    Hv, d, io = 1, 64, torch.bfloat16
    lens = [37, 100, 91]
    T = sum(lens)
    q, k, v, g = make((1, T), Hv, Hv, d, d, io, 13)
    for x in (q, k, v):
        x[0, 37:87] = float("nan")
        x[0, 87:137] = float("inf")
    cu = torch.tensor([0, 37, 137, 228], dtype=torch.int32, device=DEV)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), cu_seqlens=cu, check=True)
    for n, (a, b) in enumerate([(0, 37), (137, 228)]):
        ref = steps(q[0, a:b], k[0, a:b], v[0, a:b], g[0, a:b], torch.zeros(Hv, d, d), 1.0)
        check_prefill(o[0, a:b].cpu(), S[2 * n].cpu(), ref, io, k[0, a:b], v[0, a:b])


def test_prefill_reports_bad_offsets_and_pages(pkg):
    Hv, d, io, T = 1, 64, torch.bfloat16, 40
    q, k, v, g = (x.to(DEV) for x in make((1, T), Hv, Hv, d, d, io, 14))
    for cu in ([0, 41], [-1, 10], [0, 20, 10]):
        fin = torch.full((len(cu) - 1, Hv, d, d), 3.0, device=DEV)
        with pytest.raises(pkg.GDNError, match="index"):
            pkg.lin_prefill(q, k, v, g, final_state=fin, check=True,
                            cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
        assert bool((fin[-1] == 3).all())  # the unsound sequence, here the last, leaves no state
    cu = torch.tensor([0, 10, 30, 40], dtype=torch.int32, device=DEV)
    pool = torch.full((3, Hv, d, d), 3.0, device=DEV)
    with pytest.raises(pkg.GDNError, match="index"):
        pkg.lin_prefill(q, k, v, g, final_state=pool, cu_seqlens=cu, check=True,
                        index=torch.tensor([1, 3, 1], dtype=torch.int32, device=DEV))
    ref = steps(*(x[0, :10].cpu() for x in (q, k, v, g)), torch.zeros(Hv, d, d), 1.0)
    assert float((pool[1].cpu().double() - ref[1]).abs().max()) < 1e-3
    assert bool((pool[[0, 2]] == 3).all())


def test_prefill_strided_views(pkg):
    B, T, Hqk, Hv, d, io = 2, 70, 1, 2, 64, torch.bfloat16
    gen = torch.Generator().manual_seed(15)
    x = torch.randn(B, T, 2 * Hqk + Hv, d, generator=gen).to(io).to(DEV)
    q, k, v = x[:, :, :Hqk], x[:, :, Hqk : 2 * Hqk], x[:, :, 2 * Hqk :]
    g = (-torch.rand(Hv, T, B, generator=gen) * 0.1).to(DEV).permute(2, 1, 0)
    layers = torch.randn(B, 2, Hv, d, d, generator=gen).to(DEV)
    out = torch.zeros(B, T, 2, Hv, d, dtype=io, device=DEV)
    S0 = layers[:, 1].clone()
    o, fin = pkg.lin_prefill(q, k, v, g, layers[:, 1], out=out[:, :, 1], final_state=layers[:, 1], check=True)
    assert bool((out[:, :, 0] == 0).all())
    for b in range(B):
        ref = steps(q[b].cpu(), k[b].cpu(), v[b].cpu(), g[b].cpu(), S0[b].cpu(), 1.0)
        check_prefill(o[b].cpu(), fin[b].cpu(), ref, io, k[b].cpu(), v[b].cpu())


def test_prefill_small_f16_values_keep_the_state(pkg):
    """Values near f16's smallest normal numbers, decayed further within the chunk."""
    T, d, io = 128, 64, torch.float16
    q, k, v, g = make((1, T), 1, 1, d, d, io, 16, gmin=-0.1)
    v = (v.float() * 2.0 ** -12).to(io)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), check=True)
    check_prefill(o[0].cpu(), S[0].cpu(), steps(q[0], k[0], v[0], g[0], torch.zeros(1, d, d), 1.0), io, k[0], v[0])


def test_prefill_long_few_heads_equals_pieces(pkg):
    """A long time axis over few heads against the same tokens in two calls, and sampled rows against 64 bits."""
    T, d, io = 9000, 128, torch.bfloat16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 17, gmin=-0.02)
    x = [t.to(DEV) for t in (q, k, v, g)]
    o, S = pkg.lin_prefill(*x, scale=d ** -0.5, check=True)
    cut = 4100
    o1, S1 = pkg.lin_prefill(*(t[:, :cut] for t in x), scale=d ** -0.5, check=True)
    o2, S2 = pkg.lin_prefill(*(t[:, cut:] for t in x), S1, scale=d ** -0.5, check=True)
    ref = steps(q[0], k[0], v[0], g[0], torch.zeros(2, d, d), d ** -0.5)
    check_prefill(o[0].cpu(), S[0].cpu(), ref, io, k[0, -2000:], v[0])
    check_prefill(torch.cat([o1, o2], 1)[0].cpu(), S2[0].cpu(), ref, io, k[0, -2000:], v[0])


@pytest.mark.parametrize("T", [2048, 4097, 6000])
@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
def test_prefill_long_in_place(pkg, T, io):
    """Long enough for the time axis to be cut; the state is updated in place."""
    B, Hqk, Hv, dk, dv = 2, 1, 2, 64, 64
    q, k, v, g = make((B, T), Hqk, Hv, dk, dv, io, T, gmin=-0.05)
    S0 = torch.randn(B, Hv, dk, dv, generator=torch.Generator().manual_seed(T))
    st = S0.to(DEV)
    o, fin = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), st, scale=0.1, final_state=st, check=True)
    for b in range(B):
        ref = steps(q[b], k[b], v[b], g[b], S0[b], 0.1)
        check_prefill(o[b].cpu(), fin[b].cpu(), ref, io, k[b], v[b])


def test_prefill_long_with_pages_of_layers(pkg):
    """A cut dense batch whose states are pages of one layer of a larger pool."""
    B, T, H, d, io = 2, 2500, 2, 64, torch.bfloat16
    q, k, v, g = make((B, T), H, H, d, d, io, 40, gmin=-0.02)
    pool = torch.randn(5, 3, H, d, d, generator=torch.Generator().manual_seed(41))
    st, index = pool.to(DEV), torch.tensor([4, 1], dtype=torch.int32)
    o, fin = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), st[:, 1], scale=0.1, index=index.to(DEV), check=True)
    st = st.cpu()
    for b in range(B):
        p = int(index[b])
        ref = steps(q[b], k[b], v[b], g[b], pool[p, 1], 0.1)
        check_prefill(o[b].cpu(), st[p, 1], ref, io, k[b], v[b])
        pool[p, 1] = st[p, 1]
    assert torch.equal(st, pool)  # nothing else was written


def test_prefill_packed_long_and_short(pkg):
    """Packed sequences of which some are cut: one much longer than the rest, one of none, pages."""
    Hqk, Hv, dk, dv, io = 1, 2, 64, 128, torch.bfloat16
    lens = [100, 5000, 0, 2048, 2049, 3, 300]
    T = sum(lens)
    q, k, v, g = make((1, T), Hqk, Hv, dk, dv, io, 31, gmin=-0.05)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    pool = torch.randn(9, Hv, dk, dv, generator=torch.Generator().manual_seed(32))
    index = torch.tensor([8, 1, 3, 0, -1, 5, 2], dtype=torch.int32)
    st = pool.to(DEV)
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), st, scale=0.1, index=index.to(DEV),
                           cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV), check=True)
    o, fin = o.cpu(), st.cpu()
    for n, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        p = int(index[n])
        if a == b:
            assert torch.equal(fin[p], pool[p])
            continue
        ref = steps(q[0, a:b], k[0, a:b], v[0, a:b], g[0, a:b], pool[p] if p >= 0 else torch.zeros(Hv, dk, dv), 0.1)
        check_prefill(o[0, a:b], fin[p] if p >= 0 else ref[1], ref, io, k[0, a:b], v[0, a:b])
    assert torch.equal(fin[[4, 6, 7]], pool[[4, 6, 7]])


@pytest.mark.parametrize("B", [5, 63, 64, 65])
def test_prefill_packed_in_any_order(pkg, B):
    """More CTAs than SMs, so that sequences are taken by length: equal and empty ones, idle rows
    and unsound offsets among them; each is to the bit what a call of its own gives."""
    Hv, d, io = 32, 64, torch.bfloat16
    gen = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 300, (B,), generator=gen).tolist()
    lens[1], lens[3], lens[-1] = 0, lens[2], 299
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    T = cu[-1]
    q, k, v, g = (x.to(DEV) for x in make((1, T), 4, Hv, d, d, io, B))
    pool = torch.randn(B + 2, Hv, d, d, generator=gen).to(DEV)
    index = torch.randperm(B + 2, generator=gen)[:B].to(torch.int32)
    index[2] = -1
    st = pool.clone()
    o, _ = pkg.lin_prefill(q, k, v, g, st, index=index.to(DEV), check=True,
                           cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    want = pool.clone()
    for n in range(B):
        if lens[n]:
            a, b, p = cu[n], cu[n + 1], int(index[n])
            o1, s1 = pkg.lin_prefill(q[:, a:b], k[:, a:b], v[:, a:b], g[:, a:b], pool[p : p + 1] if p >= 0 else None,
                                     final_state=torch.empty(1, Hv, d, d, device=DEV))
            assert torch.equal(o[:, a:b], o1), n
            if p >= 0:
                want[p] = s1[0]
    assert torch.equal(st, want)
    # the last sequence's end lies behind the rows: it is reported and left out, the others stand
    cu[-1] = T + 1
    st2, o2 = pool.clone(), torch.full_like(o, 7.0)
    with pytest.raises(pkg.GDNError):
        pkg.lin_prefill(q, k, v, g, st2, index=index.to(DEV), out=o2, check=True,
                        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    want[int(index[-1])] = pool[int(index[-1])]
    assert torch.equal(st2, want)
    assert torch.equal(o2[:, : cu[-2]], o[:, : cu[-2]]) and bool((o2[:, cu[-2] :] == 7).all())


def test_prefill_packed_cut_in_any_order(pkg):
    """Longest first with one sequence cut in time."""
    Hv, d, io = 32, 64, torch.bfloat16
    lens = [70, 300, 1, 8200, 0, 300, 129]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v, g = make((1, cu[-1]), Hv, Hv, d, d, io, 41, gmin=-0.05)
    pool = torch.randn(len(lens), Hv, d, d, generator=torch.Generator().manual_seed(42))
    st = pool.to(DEV)
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), st, final_state=st, scale=0.1, check=True,
                           cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    o, fin, h = o.cpu(), st.cpu(), [0, 31]
    for n, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        if a == b:
            assert torch.equal(fin[n], pool[n])
            continue
        ref = steps(q[0, a:b, h], k[0, a:b, h], v[0, a:b, h], g[0, a:b, h], pool[n, h], 0.1)
        check_prefill(o[0, a:b, h], fin[n, h], ref, io, k[0, a:b, h], v[0, a:b, h])


def test_prefill_packed_unsound_offsets_of_long_sequences(pkg):
    """Overlapping long sequences around an unsound one: reported, nothing outside is written."""
    H, d, io, T = 1, 64, torch.bfloat16, 9000
    q, k, v, g = (x.to(DEV) for x in make((1, T), H, H, d, d, io, 33))
    cu = torch.tensor([0, 9000, 10, 9000, 20, 9000], dtype=torch.int32, device=DEV)
    fin = torch.full((5, H, d, d), 3.0, device=DEV)
    with pytest.raises(pkg.GDNError, match="index"):
        pkg.lin_prefill(q, k, v, g, final_state=fin, cu_seqlens=cu, check=True)
    assert bool((fin[[1, 3]] == 3).all())


def test_prefill_workspace_argument(pkg):
    q, k, v, g = (x.to(DEV) for x in make((1, 4096), 1, 1, 64, 64, torch.bfloat16, 34))
    want = pkg.lin_prefill(q, k, v, g, check=True)
    with pytest.raises(pkg.GDNError, match="workspace"):
        pkg.lin_prefill(q, k, v, g, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device=DEV)  # whatever it holds before
    got = pkg.lin_prefill(q, k, v, g, workspace=ws, check=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_prefill_of_few_tokens_needs_no_workspace(pkg):
    """What lets a call of few tokens go without asking for the size; a long one needs some."""
    lin = graft.submodule("lin")

    def need(T, B, H, packed):
        z = torch.zeros(B, T, H, 64, dtype=torch.bfloat16, device=DEV)
        cu = torch.zeros(9, dtype=torch.int32, device=DEV) if packed else None
        fin = torch.empty(8 if packed else B, H, 64, 64, device=DEV)
        g = torch.zeros(H, device=DEV)
        return lin._prefill_workspace(lin._prefill_args(z, z, z, g, None, fin, z, cu, None, 1.0))

    for H in (1, 2, 37, 74, 148, 149):
        for B, packed in ((1, True), (1, False), (2, False), (5, False)):
            assert need(lin._UNCUT, B, H, packed) == 0
    assert need(16384, 1, 1, True) > 0 and need(16384, 1, 1, False) > 0


def test_prefill_repeats_to_the_bit(pkg):
    x = [t.to(DEV) for t in make((2, 1500), 2, 4, 128, 128, torch.bfloat16, 35)]
    first = pkg.lin_prefill(*x, check=True)
    for _ in range(3):
        again = pkg.lin_prefill(*x)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_two_streams_at_once(pkg):
    """Two cut prefills in flight together: each has a workspace of its own."""
    sets = [[t.to(DEV) for t in make((1, 6000), 1, 2, 64, 64, torch.bfloat16, s)] for s in (36, 37)]
    want = [pkg.lin_prefill(*x, check=True) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for x, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(pkg.lin_prefill(*x))
    torch.cuda.synchronize()
    for i, (o, S) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(S, want[i % 2][1])
    pkg.check_device_status(torch.device(DEV))


def test_graph_capture_on_another_stream(pkg):
    """Prefill and decode captured together, replayed on new inputs."""
    B, T, H, d, io = 2, 200, 2, 128, torch.bfloat16
    sets = [[x.to(DEV) for x in make((B, T), H, H, d, d, io, s)] for s in (20, 21)]
    tok = [[x.to(DEV) for x in make((B,), H, H, d, d, io, s)] for s in (22, 23)]
    x, y = [t.clone() for t in sets[0]], [t.clone() for t in tok[0]]
    st = torch.empty(B, H, d, d, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pkg.lin_prefill(*x, final_state=st)
        pkg.lin_decode(*y, st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        o, _ = pkg.lin_prefill(*x, final_state=st)
        od = pkg.lin_decode(*y, st)
    for i in (1, 0):
        for a, b in zip(x + y, sets[i] + tok[i]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want, S = pkg.lin_prefill(*sets[i])
        want_d = pkg.lin_decode(*tok[i], S)
        assert torch.equal(o, want) and torch.equal(od, want_d) and torch.equal(st, S)
    pkg.check_device_status(torch.device(DEV))


def check_finite_part(o, S, ref, io, k, v):
    """What is finite by the definition is so here, and close; the rest is not."""
    ro, rS, oa, Sa = ref
    assert torch.equal(torch.isfinite(o), torch.isfinite(ro)) and torch.equal(torch.isfinite(S), torch.isfinite(rS))
    fo, fS = torch.isfinite(ro), torch.isfinite(rS)
    zero = torch.zeros((), dtype=torch.float64)
    k, v = torch.nan_to_num(k.float(), 0, 0, 0), torch.nan_to_num(v.float(), 0, 0, 0)
    check_prefill(torch.where(fo, o.double(), zero), torch.where(fS, S.double(), zero),
                  (torch.where(fo, ro, zero), torch.where(fS, rS, zero), torch.where(fo, oa, zero),
                   torch.where(fS, Sa, zero)), io, k, v)


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 192)])
@pytest.mark.parametrize("gmin", [-0.2, -2.0, -30.0])
def test_prefill_values_that_are_not_finite_reach_no_earlier_row(pkg, gmin, dk, dv, io):
    T, inf, nan = 300, float("inf"), float("nan")
    q, k, v, g = make((1, T), 1, 2, dk, dv, io, 50, gmin=gmin)
    S0 = torch.randn(1, 2, dk, dv, generator=torch.Generator().manual_seed(51))
    q[0, 70, 0, 3] = nan  # its own row alone
    for t, h, c, x in [(5, 0, 0, inf), (5, 0, 33, nan), (64, 0, 7, -inf), (127, 0, 40, nan), (127, 1, 1, inf), (128, 1, 2, nan),
                       (200, 1, 63, inf), (130, 1, 62, nan), (299, 0, dv - 1, nan), (3, 1, 62, inf)]:
        v[0, t, h, c] = x
    args = [x.to(DEV) for x in (q, k, v, g)]
    o, S = pkg.lin_prefill(*args, S0.to(DEV), scale=0.1, check=True)
    check_finite_part(o[0].cpu(), S[0].cpu(), steps(q[0], k[0], v[0], g[0], S0[0], 0.1), io, k[0], v[0])
    k[0, 250, 0, 5] = -inf
    o, S = pkg.lin_prefill(args[0], k.to(DEV), *args[2:], S0.to(DEV), scale=0.1, check=True)
    check_finite_part(o[0].cpu(), S[0].cpu(), steps(q[0], k[0], v[0], g[0], S0[0], 0.1), io, k[0], v[0])


def test_prefill_padded_batch(pkg):
    """Sequences of a dense batch that end early, with whatever behind them: their rows are those of the sequence alone."""
    T, H, d, io = 260, 2, 128, torch.bfloat16
    q, k, v, g = make((3, T), H, H, d, d, io, 52)
    lens = [1, 150, 250]
    for b, n in enumerate(lens):
        for x in (q, k, v):
            x[b, n:] = float("nan")
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), check=True)
    for b, n in enumerate(lens):
        ref = steps(q[b, :n], k[b, :n], v[b, :n], g[b, :n], torch.zeros(H, d, d), 1.0)
        check_prefill(o[b, :n].cpu(), ref[1], ref, io, k[b, :n], v[b, :n])


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gmin", [-0.2, -2.0, -30.0])
@pytest.mark.parametrize("at", [0, 40, 127, 200])
def test_prefill_nan_gate_reaches_no_earlier_row(pkg, at, gmin, io):
    T, d = 220, 64
    q, k, v, g = make((1, T), 1, 2, d, d, io, 53, gmin=gmin)
    g[0, at, 1] = float("nan")
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), scale=0.1, check=True)
    check_finite_part(o[0].cpu(), S[0].cpu(), steps(q[0], k[0], v[0], g[0], torch.zeros(2, d, d), 0.1), io, k[0], v[0])


@pytest.mark.parametrize("gmin", [-0.4, -0.8, -1.6, -3.0])
def test_prefill_small_states(pkg, gmin):
    """States and values of 2^-60 keep their relative precision."""
    T, d, io = 200, 64, torch.bfloat16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 54, gmin=gmin)
    S0 = torch.randn(1, 2, d, d, generator=torch.Generator().manual_seed(55)) * 2.0 ** -60
    v = (v.float() * 2.0 ** -60).to(io)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), check=True)
    ro, rS, oa, Sa = steps(q[0], k[0], v[0], g[0], S0[0], 1.0)
    u = half_step(io)
    # below 2^-126, the smallest normal number of bf16 and fp32, nothing is promised
    tol = u * ro.abs() + (u + 2 * W + 64 * E) * oa + 2.0 ** -126
    # the rows that decay leaves less than 2^-80 of the state before their chunk take that much
    for c in range(0, T, 128):
        at = steps(q[0, :c], k[0, :c], v[0, :c], g[0, :c], S0[0], 1.0)[3] if c else S0[0].double().abs()
        rows = slice(c, min(c + 128, T))
        tol[rows] += 2.0 ** -80 * torch.einsum("td,hde->the", q[0, rows, 0].double().abs(), at)
    assert bool(((o[0].cpu().double() - ro).abs() <= tol).all())
    assert bool(((S[0].cpu().double() - rS).abs() <= (u * u + 64 * E) * Sa + 2.0 ** -126).all())


@pytest.mark.parametrize("gmin", [-0.5, -1.0, -1.4, -2.5])
@pytest.mark.parametrize("scale", [2.0 ** -24 * 1.3, -(2.0 ** -9), 2.0 ** 20])
def test_prefill_large_values_at_any_scale(pkg, scale, gmin):
    """Outputs of up to 2^43 or so, whatever part of that the scale is."""
    T, d, io = 300, 64, torch.bfloat16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 56, gmin=gmin)
    v = (v.float() * 2.0 ** 36 / abs(scale)).to(io)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), scale=scale, check=True)
    ro, rS, oa, Sa = steps(q[0], k[0], v[0], g[0], torch.zeros(2, d, d), scale)
    for c in range(128, T, 128):  # a row takes 2^-80 of the state before its chunk where decay leaves less
        at = steps(q[0, :c], k[0, :c], v[0, :c], g[0, :c], torch.zeros(2, d, d), scale)[3]
        rows = slice(c, min(c + 128, T))
        oa[rows] += abs(scale) * 2.0 ** -80 / (half_step(io) + 2 * W) * torch.einsum("td,hde->the", q[0, rows, 0].double().abs(), at)
    check_prefill(o[0].cpu(), S[0].cpu(), (ro, rS, oa, Sa), io, k[0], v[0])


def test_prefill_scale_of_zero(pkg):
    q, k, v, g = (x.to(DEV) for x in make((1, 200), 1, 2, 64, 64, torch.bfloat16, 57))
    o, S = pkg.lin_prefill(q, k, v, g, scale=0.0, check=True)
    assert bool((o == 0).all()) and torch.equal(S, pkg.lin_prefill(q, k, v, g)[1])


@pytest.mark.parametrize("early,late,gmin", [(1000.0, 1e-3, -0.25), (6e4, 1e-4, -0.2), (1.0, 0.0, -0.4), (2.0 ** -14, 2.0 ** -20, -0.1),
                                             (2.0 ** -24, 2.0 ** -24, 0.0), (1.0, 1.0, -0.2), (6e4, 6e4, 0.0)])
def test_prefill_f16_state_of_uneven_values(pkg, early, late, gmin):
    """Large values that have decayed by the chunk's end beside small ones, and values near f16's ends.  What is
    left of the two parts of a term is u^2 of it, and 2^-39 of its column's largest in the chunk, 128 times."""
    T, dk, dv, io = 256, 64, 128, torch.float16
    q, k, v, g = make((1, T), 1, 2, dk, dv, io, 58, gmin=gmin)
    size = torch.where(torch.arange(T) % 128 < 20, early, late)[:, None, None]
    v = (torch.rand(T, 2, dv, generator=torch.Generator().manual_seed(59)) * 2 - 1) * size
    v[:, :, 1::2] *= 2.0 ** -8  # columns next to one another differ too
    v = v.to(io)[None]
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), scale=2.0 ** -7, check=True)
    _, rS, _, Sa = steps(q[0], k[0], v[0], g[0], torch.zeros(2, dk, dv), 2.0 ** -7)
    u = half_step(io)
    tol = (u * u + 64 * E) * Sa + 2.0 ** -32 * Sa.amax(1, keepdim=True)
    assert bool(((S[0].cpu().double() - rS).abs() <= tol).all()), float(((S[0].cpu().double() - rS).abs() / tol).max())


def test_prefill_f16_growing_gates_keep_the_state(pkg):
    """Weights e^(G_C - G_j) far beyond f16's range."""
    T, d, io = 200, 64, torch.float16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 60, gmin=0.5)
    v = (v.float() * 2.0 ** -10).to(io)
    _, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), check=True)
    _, rS, _, Sa = steps(q[0], k[0], v[0], g[0], torch.zeros(2, d, d), 1.0)
    u = half_step(io)
    assert float(rS.abs().max()) > 2.0 ** 40
    assert bool(((S[0].cpu().double() - rS).abs() <= (u * u + 64 * E) * Sa + 2.0 ** -32 * Sa.amax(1, keepdim=True)).all())


def check_f16_rows(o, ref, v):
    """f16 I/O: the output's rounding, and that of P or of the state that the queries meet, tf32 (u each, of their
    terms); a scaled P below 2^-14 is off by at most 2^-25 (of the unscaled, a little more: hence 2^-16)."""
    ro, _, oa, _ = ref
    u = half_step(torch.float16)
    tol = u * ro.abs() + 2.0 ** -25 + (u + 2.0 ** -16 + 64 * E) * oa + 2.0 ** -25 * 128 * v.double().abs().amax()
    assert bool(((o.double() - ro).abs() <= tol).all()), float(((o.double() - ro).abs() / tol).max())


@pytest.mark.parametrize("dk,dv", [(64, 64), (64, 128), (128, 64), (128, 128), (128, 192)])
@pytest.mark.parametrize("T,gmin", [(1, -0.2), (130, 0.0), (257, -0.05), (400, -0.5), (400, -2.0)])
def test_prefill_f16_outputs(pkg, T, gmin, dk, dv):
    """Queries and states are not held in bf16 alone where the I/O is f16."""
    io = torch.float16
    q, k, v, g = make((1, T), 1, 2, dk, dv, io, 61, gmin=gmin)
    S0 = torch.randn(1, 2, dk, dv, generator=torch.Generator().manual_seed(62)) * 30
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=0.05, check=True)
    ref = steps(q[0], k[0], v[0], g[0], S0[0], 0.05)
    check_f16_rows(o[0].cpu(), ref, v)
    check_prefill(o[0].cpu(), S[0].cpu(), ref, io, k[0], v[0])


def test_prefill_f16_states_beyond_its_range(pkg):
    """A state that f16 does not hold, queries that make its outputs small."""
    T, d, io = 200, 128, torch.float16
    q, k, v, g = make((1, T), 1, 1, d, d, io, 63, gmin=-0.01)
    S0 = torch.randn(1, 1, d, d, generator=torch.Generator().manual_seed(64)) * 1e7
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=2.0 ** -15, check=True)
    check_f16_rows(o[0].cpu(), steps(q[0], k[0], v[0], g[0], S0[0], 2.0 ** -15), v)


@pytest.mark.parametrize("T", [5000, 9000])
def test_prefill_f16_long(pkg, T):
    """Cut in time, and sequences of many chunks, at the shape whose K has one stage."""
    d, io = 128, torch.float16
    q, k, v, g = make((1, T), 1, 2, d, d, io, T, gmin=-0.02)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), scale=d ** -0.5, check=True)
    ref = steps(q[0], k[0], v[0], g[0], torch.zeros(2, d, d), d ** -0.5)
    check_f16_rows(o[0].cpu(), ref, v)
    check_prefill(o[0].cpu(), S[0].cpu(), ref, io, k[0, -2000:], v[0])


def f16_size(x, most):
    return (x / x.abs().max() * most).to(torch.float16)


def check_f16_range(o, ref):
    """check_f16_rows where P passes f16's range: its terms below 2^-39 of the row's largest may be lost, 128 of them;
    no value of v is much larger than those that the row's largest scores meet, hence 2^-30 of the sum."""
    ro, _, oa, _ = ref
    u = half_step(torch.float16)
    fits = ro.abs() < 65000
    assert float(fits.double().mean()) > 0.9
    tol = u * ro.abs() + 2.0 ** -25 + (u + 2.0 ** -16 + 64 * E) * oa + 2.0 ** -30 * oa.amax(2, keepdim=True)
    assert bool(((o.double() - ro).abs() <= tol)[fits].all()), float(((o.double() - ro).abs() / tol)[fits].max())


@pytest.mark.parametrize("scale,vmax", [(1.0, 2.0 ** -20), (2.0 ** 40, 0.0), (2.0 ** -30, 1.0), (2.0 ** -45, 6e4), (-(2.0 ** -60), 6e4)])
@pytest.mark.parametrize("gmin", [0.0, -0.2, -2.0])
def test_prefill_f16_scores_beyond_its_range(pkg, gmin, scale, vmax):
    """Queries and keys near f16's largest: scores of up to 2^71, with outputs that f16 holds; and scores so small
    that f16 would hold none of them."""
    T, d, io = 200, 64, torch.float16
    gen = torch.Generator().manual_seed(65)
    q, k = (f16_size(torch.randn(1, T, 1, d, generator=gen), 6e4) for _ in range(2))
    v = f16_size(torch.randn(1, T, 2, d, generator=gen), max(vmax, 2.0 ** -24)) * (vmax > 0)
    g = torch.rand(1, T, 2, generator=gen) * gmin
    S0 = torch.randn(1, 2, d, d, generator=gen) * 2.0 ** -20 / scale * (vmax == 0)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=scale, check=True)
    ref = steps(q[0], k[0], v[0], g[0], S0[0], scale)
    check_f16_range(o[0].cpu(), ref)
    u = half_step(io)
    # (2^-126, fp32's smallest normal number: a state of 2^-60 that decays by 2^-288 is none of fp32's)
    tol = (u * u + 64 * E) * ref[3] + 2.0 ** -32 * ref[3].amax(1, keepdim=True) + 2.0 ** -126
    assert bool(((S[0].cpu().double() - ref[1]).abs() <= tol).all())


def test_prefill_f16_growing_gates(pkg):
    """Scores that growing gates take beyond f16's range, with outputs inside it."""
    T, d, io = 120, 64, torch.float16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 66, gmin=0.25)
    v = (v.float() * 2.0 ** -18).to(io)
    v[:, 8:] = 0
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), check=True)
    check_f16_range(o[0].cpu(), steps(q[0], k[0], v[0], g[0], torch.zeros(2, d, d), 1.0))


@pytest.mark.parametrize("scale", [2.0 ** 100, 2.0 ** -100, 0.0])
def test_prefill_f16_rows_without_scores(pkg, scale):
    """Keys of zero: only the state before is read, at any scale."""
    T, d, io = 140, 64, torch.float16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 67, gmin=-0.1)
    k[:] = 0
    S0 = torch.randn(1, 2, d, d, generator=torch.Generator().manual_seed(68)) / (scale or 1.0)
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=scale, check=True)
    ref = steps(q[0], k[0], v[0], g[0], S0[0], scale)
    check_f16_range(o[0].cpu(), ref)
    assert bool(((S[0].cpu().double() - ref[1]).abs() <= 64 * E * ref[3] + 2.0 ** -126).all())  # (fp32's smallest)


def test_axes_of_one_entry_have_any_stride(pkg):
    """What torch calls contiguous: [1, T, 1, d] and [1, 1, d] with strides of 1."""
    T, d, io = 10, 64, torch.bfloat16
    q, k, v, g = (x.to(DEV) for x in make((1, T), 1, 1, d, d, io, 69))
    odd = [x.as_strided(x.shape, (T * d, d, 1, 1)) for x in (q, k, v)]
    assert odd[0].stride() == (T * d, d, 1, 1) and odd[0].is_contiguous()
    want, S = pkg.lin_prefill(q, k, v, g, check=True)
    wide = torch.zeros(1, 1, d, d + 1, device=DEV)[..., :d]  # (not contiguous: refused)
    with pytest.raises(pkg.GDNError):
        pkg.lin_prefill(*odd, g, final_state=wide)
    fin = torch.empty(d * d + 3, device=DEV)[: d * d].as_strided((1, 1, d, d), (1, 1, d, 1))
    got, _ = pkg.lin_prefill(*odd, g, final_state=fin, check=True)
    assert torch.equal(got, want) and torch.equal(fin, S)
    q, k, v = (x[:, 0].clone() for x in (q, k, v))
    want = pkg.lin_decode(q, k, v, g[:, 0], S, check=True)
    q, k, v = (x.as_strided((1, 1, d), (1, 1, 1)) for x in (q, k, v))
    assert torch.equal(pkg.lin_decode(q, k, v, g[:, 0], fin, check=True), want) and torch.equal(fin, S)


def test_states_of_one_layer_into_another(pkg):
    """Layers of one tensor, whose pages lie between one another: out of place, with nothing else written."""
    B, T, H, d, io = 3, 70, 2, 64, torch.bfloat16
    layers = torch.randn(B, 3, H, d, d, generator=torch.Generator().manual_seed(70)).to(DEV)
    before = layers.clone()
    q, k, v, g = (x.to(DEV) for x in make((B, T), H, H, d, d, io, 71))
    o, S = pkg.lin_prefill(q, k, v, g, layers[:, 0].clone(), check=True)
    got, _ = pkg.lin_prefill(q, k, v, g, layers[:, 0], final_state=layers[:, 2], check=True)
    assert torch.equal(got, o) and torch.equal(layers[:, 2], S) and torch.equal(layers[:, :2], before[:, :2])
    token = [x[:, 0].contiguous() for x in (q, k, v, g)]
    want = S.clone()
    o = pkg.lin_decode(*token, want)
    assert torch.equal(pkg.lin_decode(*token, layers[:, 2], state_out=layers[:, 1], check=True), o)
    assert torch.equal(layers[:, 1], want) and torch.equal(layers[:, 2], S) and torch.equal(layers[:, 0], before[:, 0])


def test_prefill_refuses_offsets_of_no_sequence(pkg):
    q, k, v, g = (x.to(DEV) for x in make((1, 5), 1, 1, 64, 64, torch.bfloat16, 72))
    for cu in (torch.empty(0), torch.zeros(1), torch.tensor(0)):
        with pytest.raises(pkg.GDNError, match="cu_seqlens"):
            pkg.lin_prefill(q, k, v, g, cu_seqlens=cu.to(torch.int32).to(DEV))


@pytest.mark.parametrize("rise", [0.01, 3.0])
@pytest.mark.parametrize("gmin", [-0.5, -2.0, -30.0])
def test_prefill_f16_a_gate_that_grows_among_falling_ones(pkg, gmin, rise):
    T, d, io = 200, 64, torch.float16
    q, k, v, g = make((1, T), 1, 2, d, d, io, 73, gmin=gmin)
    g[0, [3, 70, 71, 127, 190]] = rise
    S0 = torch.randn(1, 2, d, d, generator=torch.Generator().manual_seed(74))
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=0.1, check=True)
    ref = steps(q[0], k[0], v[0], g[0], S0[0], 0.1)
    check_f16_rows(o[0].cpu(), ref, v)
    check_prefill(o[0].cpu(), S[0].cpu(), ref, io, k[0], v[0])


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gmin", [-0.5, -1.5, -3.0, -30.0])
def test_prefill_keys_of_zero_at_a_large_scale(pkg, gmin, io):
    """No decay times the scale may pass fp32 on the way to a product with zero."""
    T, d, scale = 140, 64, 2.0 ** 100
    q, k, v, g = make((1, T), 1, 2, d, d, io, 75, gmin=gmin)
    k[:] = 0
    S0 = torch.randn(1, 2, d, d, generator=torch.Generator().manual_seed(76)) / scale
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), scale=scale, check=True)
    ro, _, oa, _ = steps(q[0], k[0], v[0], g[0], S0[0], scale)
    u = half_step(io)
    # a row takes 2^-80 of the state before its chunk where decay leaves less
    at = scale * torch.einsum("td,hde->the", q[0, :, 0].double().abs(), S0[0].double().abs())
    # the state itself, of 2^-100 and decaying, comes below fp32's smallest normal number, where its steps are 2^-149
    # wide: each of its entries may be off by one, and scale |q| of them make the output
    at += scale * 2.0 ** (80 - 149) * q[0].double().abs().sum(-1, keepdim=True)
    tol = u * ro.abs() + (u + 2 * W + 64 * E) * oa + 2.0 ** -80 * at + (2.0 ** -25 if io == torch.float16 else 2.0 ** -126)
    assert bool(((o[0].cpu().double() - ro).abs() <= tol).all())


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
def test_prefill_packed_long_pages_and_values_that_are_not_finite(pkg, io):
    """Cut and whole sequences side by side, some of them with values that are not finite: those stay where they are."""
    Hv, dk, dv = 2, 128, 128
    lens = [100, 9000, 0, 2049, 300, 1]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    q, k, v, g = make((1, cu[-1]), 1, Hv, dk, dv, io, 77, gmin=-0.05)
    v[0, cu[1] + 8000, 0, 5] = float("nan")
    v[0, cu[3] + 1000, 1, 127] = float("inf")
    k[0, cu[4] + 299, 0, 0] = float("nan")
    g[0, cu[3] - 1, 0] = float("-inf")
    pool = torch.randn(8, Hv, dk, dv, generator=torch.Generator().manual_seed(78))
    index = torch.tensor([7, 0, 3, 5, 1, 2], dtype=torch.int32)
    st = pool.to(DEV)
    o, _ = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), st, scale=0.1, index=index.to(DEV), check=True,
                           cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=DEV))
    o, fin = o.cpu(), st.cpu()
    for n, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        p = int(index[n])
        if a == b:
            assert torch.equal(fin[p], pool[p])
            continue
        ref = steps(q[0, a:b], k[0, a:b], v[0, a:b], g[0, a:b], pool[p], 0.1)
        check_finite_part(o[0, a:b], fin[p], ref, io, k[0, a:b], v[0, a:b])
    assert torch.equal(fin[[4, 6]], pool[[4, 6]])


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
def test_prefill_captured_and_on_two_streams(pkg, io):
    """Replays on new inputs, and two calls in flight, give what single calls do, to the bit."""
    sets = [[x.to(DEV) for x in make((2, 300), 1, 2, 128, 128, io, s)] for s in (79, 80)]
    want = [pkg.lin_prefill(*x, check=True) for x in sets]
    x = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, S = pkg.lin_prefill(*x)
    streams = [torch.cuda.Stream() for _ in sets]
    for i in (1, 0):
        for a, b in zip(x, sets[i]):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        got = []
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got.append(pkg.lin_prefill(*sets[j]))
        torch.cuda.synchronize()
        assert torch.equal(o, want[i][0]) and torch.equal(S, want[i][1])
        assert all(torch.equal(a, b) for g1, w in zip(got, want) for a, b in zip(g1, w))
    pkg.check_device_status(torch.device(DEV))


@pytest.mark.parametrize("io", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("at", [0, 64, 96, 128])
def test_prefill_reset_drops_a_state_of_any_size(pkg, at, io):
    """A page that holds whatever was there before, and a decay of zero at the start of a chunk or of a block in it."""
    T, d = 200, 64
    q, k, v, g = make((1, T), 1, 2, d, d, io, 81, gmin=-0.1)
    g[0, at] = float("-inf")
    S0 = torch.randn(1, 2, d, d, generator=torch.Generator().manual_seed(82)) * 1e30
    o, S = pkg.lin_prefill(*(x.to(DEV) for x in (q, k, v, g)), S0.to(DEV), check=True)
    ro, rS, oa, Sa = steps(q[0], k[0], v[0], g[0], S0[0], 1.0)
    check_prefill(o[0, at:].cpu(), S[0].cpu(), (ro[at:], rS, oa[at:], Sa), io, k[0], v[0])
