"""AdamW over many tensors (states in 32 and in 8 bits) and the global gradient norm,
against the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32, relative):
  m' = m + (x - m) w1, x = g c: the roundings of x, x - m, w1, the product and the sum are each
       at most u (|m| + |x|): 5 u (|m| + |x|).
  v' = v b2 + x x w2, all terms >= 0: x x carries 2 u of x and u of its own, w2 and the product
       u each; v b2 carries 2 u; the sum u: 6 u v'.
  r' = sqrt(v'): half of that and its own u: 4 u r'.
  d  = r' inv + eps: r's 4 u, u each for inv, the product, eps and the sum: 8 u d.
  p' = p decay + (m'/d) step: 3 u |p| for the first term and its place in the sum; the update
       carries |m' error| step / d, and 8 u (d) + 2 u (the reciprocal's 1 ulp) + u (product
       with m') + u (step) + u (product) + u (sum) = 14 u of itself.
e4m3 codes are rounded to one of the two neighbours: less than one step, 2^-3 of the value's
power of two, 2^-9 of the scale below 2^-6 of it."""
import ctypes
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
M32 = 0xFFFFFFFF


# ------------------------------------------------------------------ plain forms
def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _words(n, seed, step, ordinal):
    key = _mix((_mix((_mix((_mix(seed & M32) + (seed >> 32)) & M32) + step) & M32) + ordinal) & M32)
    i = torch.arange(n, dtype=torch.int64)
    return _mix(((i & M32) * 0x9E3779B9 + (i >> 32) * 0x3C6EF373 + key) & M32)


def _scale_bytes(x, slack=0.0):
    """The scale bytes of x's blocks of 64, from the definition in 64 bits."""
    x = torch.where(torch.isfinite(x), x.abs(), 0.0).double() * (1 + slack)
    x = torch.nn.functional.pad(x, (0, -x.numel() % 64)).view(-1, 64).amax(1)
    e = torch.frexp(x)[1] - 1  # x in [2^e, 2^(e+1))
    return torch.where(x > 0, (e - 7 + 127).clamp_min(0), 0).to(torch.int64)


def _values(codes, scale):
    b = scale.view(torch.uint8).to(torch.float64)
    return codes.reshape(-1).to(torch.float64) * torch.exp2(b - 127).repeat_interleave(64)[:codes.numel()]


def _step_of(x, bytes_):
    """One e4m3 step at x (64 bits) under the scales."""
    s = torch.exp2(bytes_.double() - 127).repeat_interleave(64)[:x.numel()]
    e = torch.frexp(x.abs() / s)[1] - 1
    return s * torch.exp2(torch.clamp_min(e.double(), -6.0) - 3)


def _exact(p, g, m, v, lr, wd, t, c=1.0, betas=(0.9, 0.999), eps=1e-15):
    """(p', m', v') in 64 bits and the bounds of their fp32 errors."""
    p, g, m, v = (x.double().reshape(-1) for x in (p, g, m, v))
    b1, b2 = betas
    x = g * c
    m2, v2 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    d = (v2 / (1 - b2 ** t)).sqrt() + eps
    k = lr / (1 - b1 ** t)
    up = k * m2 / d
    em = 5 * U * (m.abs() + x.abs())
    return (p * (1 - lr * wd) - up, m2, v2), (3 * U * p.abs() + k * em / d + 14 * U * up.abs(), em, 6 * U * v2)


def _within(got, want, bound, what):
    got = got.detach().cpu().double().reshape(-1)
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float(((got - want).abs() / bound.clamp_min(1e-300)).max()):.2f} bounds")


def _inputs(n, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda: torch.randn(n, generator=g)  # noqa: E731
    grad = r() * torch.exp(2 * r()) * 1e-6 * (torch.rand(n, generator=g) < 0.7)
    m = r() * torch.exp(r()) * 1e-6
    v = (m * m + 1e-16) * torch.exp(2 * r())
    return r().to(dtype), grad.to(dtype), m, v


def _state8(m, v, dev):
    """An 8-bit state near m and sqrt(v): codes from torch's own cast, to nearest."""
    st = {"step": 0}
    for k, x in (("exp_avg", m), ("exp_rms", v.sqrt())):
        b = _scale_bytes(x)
        s = torch.exp2(b.double() - 127).repeat_interleave(64)[:x.numel()]
        q = (x.double().reshape(-1) / s).float()
        codes = q.to(torch.float8_e4m3fn)
        st[k] = codes.view(x.shape).to(dev)
        st[k + "_scale"] = b.to(torch.uint8).view(torch.float8_e8m0fnu).to(dev)
    return st


# ------------------------------------------------------------------ CPU: refusals
@pytest.fixture(scope="module")
def lib():
    from diff_gaussian_rasterization import _C

    return _C.load_library()


def _err(lib):
    return lib.gsr_last_error().decode()


def test_adamw_abi_refusals(lib):
    from diff_gaussian_rasterization import _C

    S = _C.GsrAdamWSegment
    assert ctypes.sizeof(S) == 6 * 8 + 3 * 8 + 8
    call = lambda segs, n=None, dt=0, bits=32, b1=0.9, b2=0.999, eps=0.0: lib.gsr_adamw_step(  # noqa: E731
        (S * max(1, len(segs)))(*segs), len(segs) if n is None else n, dt, bits, b1, b2, eps, None, 0, None)
    ok = (1, 1, 1, 1, None, None, 4, 0.1, 0.0, 1, 0)
    assert call([ok], n=-1) != 0 and "segment list" in _err(lib)
    assert lib.gsr_adamw_step(None, 1, 0, 32, 0.9, 0.999, 0.0, None, 0, None) != 0
    assert call([ok], dt=2) != 0 and "dtype" in _err(lib)
    assert call([ok], bits=16) != 0 and "state_bits" in _err(lib)
    assert call([ok], b1=1.0) != 0 and "betas" in _err(lib)
    assert call([ok], b2=math.nan) != 0 and "betas" in _err(lib)
    assert call([ok], eps=-1.0) != 0
    assert call([ok], eps=1e-40) != 0 and "eps" in _err(lib)  # the reciprocal takes normal numbers
    assert call([ok[:9] + (0, 0)]) != 0 and "step" in _err(lib)
    assert call([ok[:6] + (-1,) + ok[7:]]) != 0 and "size" in _err(lib)
    assert call([ok[:6] + ((1 << 33) + 1,) + ok[7:]]) != 0 and "size" in _err(lib)
    assert call([(None,) + ok[1:]]) != 0 and "NULL" in _err(lib)
    assert call([ok], bits=8) != 0 and "NULL" in _err(lib)  # no scales
    # nothing to do is not an error
    assert call([], n=0) == 0
    assert call([(None,) * 6 + (0, 0.1, 0.0, 1, 0)] * 3) == 0


def test_grad_norm_abi_refusals(lib):
    from diff_gaussian_rasterization import _C

    S = _C.GsrGradSegment
    assert ctypes.sizeof(S) == 24
    call = lambda seg, mx=1.0, scratch=1, out=1: lib.gsr_grad_norm((S * 1)(seg), 1, mx, scratch, out, None)  # noqa: E731
    assert call((1, 4, 0, 0), mx=math.nan) != 0 and "max_norm" in _err(lib)
    assert call((1, 4, 0, 0), mx=-1.0) != 0
    assert call((1, 4, 0, 0), scratch=None) != 0 and "NULL" in _err(lib)
    assert call((1, -4, 0, 0)) != 0 and "size" in _err(lib)
    assert call((1, 4, 7, 0)) != 0 and "dtype" in _err(lib)
    assert call((None, 4, 0, 0)) != 0 and "NULL" in _err(lib)
    assert lib.gsr_grad_norm(None, 1, 1.0, 1, 1, None) != 0
    assert lib.gsr_grad_norm_scratch_bytes(1) >= 8 * 1024
    assert lib.gsr_grad_norm_scratch_bytes(129) >= 2 * 8 * 1024


def test_python_refusals_on_cpu():
    import train_ops

    p = torch.zeros(5)
    st = train_ops.adamw_state(p)
    with pytest.raises(RuntimeError, match="GPU"):
        train_ops.adamw_step([p], [p.clone()], [st], 0.1)
    assert st["step"] == 0
    with pytest.raises(ValueError, match="gradients"):
        train_ops.adamw_step([p], [], [st], 0.1)
    with pytest.raises(ValueError, match="lr"):
        train_ops.adamw_step([p], [p], [st], [0.1, 0.2])
    with pytest.raises(RuntimeError, match="GPU"):
        train_ops.grad_norm([p])
    with pytest.raises(ValueError, match="no gradients"):
        train_ops.grad_norm([])
    with pytest.raises(ValueError, match="state_bits"):
        train_ops.adamw_state(p, 16)
    with pytest.raises(ValueError, match="state_bits"):
        train_ops.FusedAdamW([{"params": [p]}], state_bits=4)
    train_ops.adamw_step([], [], [], 0.1)
    train_ops.FusedAdamW([{"params": [p]}]).step()  # no gradients: nothing to do


def test_state8_layout_and_values_on_cpu():
    import train_ops

    st = train_ops.adamw_state(torch.zeros(13, 5), 8)
    assert st["exp_avg"].shape == (13, 5) and st["exp_avg_scale"].numel() == 2
    assert not train_ops.unpack_state8(st["exp_avg"], st["exp_avg_scale"]).any()
    codes = torch.arange(0x78, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scale = torch.tensor([0, 130], dtype=torch.uint8).view(torch.float8_e8m0fnu)
    got = train_ops.unpack_state8(codes, scale)
    torch.testing.assert_close(got.double(), _values(codes, scale), rtol=0, atol=0)


def test_train_state_refuses_adamw_options_without_fused():
    import synthetic
    import train_step

    g = synthetic.make_gaussians(4, 0)
    with pytest.raises(ValueError, match="fused"):
        train_step.TrainState(g, 1.0, state_bits=8)


# ------------------------------------------------------------------ GPU: the step
SIZES = [1, 3, 63, 64, 65, 1023, 1024, 1025, 4097, 20_011]


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_step32_against_64_bits(dev, wd, clip):
    import train_ops

    ins = [_inputs(n, n) for n in SIZES]
    steps = [3 * k for k in range(len(SIZES))]  # each tensor counts its own
    lrs = [10.0 ** -(1 + k % 4) for k in range(len(SIZES))]
    P, G = [i[0].to(dev) for i in ins], [i[1].to(dev) for i in ins]
    st = [{"step": t, "exp_avg": i[2].to(dev), "exp_avg_sq": i[3].to(dev)} for i, t in zip(ins, steps)]
    c, scale = 1.0, None
    if clip:
        norm, scale = train_ops.grad_norm(G, 1e-6)
        c = float(scale)
        assert 0 < c < 1
    train_ops.adamw_step(P, G, st, lrs, wd, grad_scale=scale)
    for k, (p, g, m, v) in enumerate(ins):
        want, bound = _exact(p, g, m, v, lrs[k], wd, steps[k] + 1, c)
        assert st[k]["step"] == steps[k] + 1
        for got, w, b, what in zip((P[k], st[k]["exp_avg"], st[k]["exp_avg_sq"]), want, bound, "pmv"):
            _within(got, w, b, f"n={SIZES[k]} {what}")


@pytest.mark.gpu
def test_step32_follows_torch_adamw(dev):
    """Ten steps beside torch.optim.AdamW (its order of operations up to one reciprocal)."""
    import train_ops

    shapes, lrs = [(1000, 3), (1000, 15, 3), (1000, 0, 3), (1000, 1), (333, 4)], [1e-3, 1e-4, 1e-4, 5e-2, 1e-3]
    g = torch.Generator().manual_seed(0)
    base = [torch.randn(s, generator=g) for s in shapes]
    pa = [b.clone().to(dev).requires_grad_(True) for b in base]
    pb = [b.clone().to(dev).requires_grad_(True) for b in base]
    mk = lambda ps: [{"params": [p], "lr": lr} for p, lr in zip(ps, lrs)]  # noqa: E731
    fa = train_ops.FusedAdamW(mk(pa), eps=1e-8, weight_decay=0.02, max_norm=30.0)
    ta = torch.optim.AdamW(mk(pb), eps=1e-8, weight_decay=0.02)
    for _ in range(10):
        for p, q in zip(pa, pb):
            p.grad = torch.randn(p.shape, generator=g).to(dev)
            q.grad = p.grad.clone()
        fa.step()
        norm = torch.nn.utils.clip_grad_norm_(pb, 30.0)
        torch.testing.assert_close(fa.grad_norm, norm, rtol=1e-5, atol=0)
        ta.step()
    for p, q in zip(pa, pb):
        # ten steps of about 12 roundings each, of updates and parameters of order 1
        torch.testing.assert_close(p, q, rtol=2e-5, atol=2e-6)
        torch.testing.assert_close(fa.state[p]["exp_avg"], ta.state[q]["exp_avg"], rtol=2e-5, atol=2e-6)
        torch.testing.assert_close(fa.state[p]["exp_avg_sq"], ta.state[q]["exp_avg_sq"], rtol=2e-5, atol=1e-9)


def _plain8(p, g, m, r, lr, wd, t, words, c=1.0, betas=(0.9, 0.999), eps=1e-15):
    """The 8-bit step in fp32 torch operations on the CPU, each of which rounds once: the codes."""
    b1, b2 = betas
    x = g.float() * c
    m2 = m + (x - m) * (1.0 - b1)
    v2 = (r * r) * b2 + (x * x) * (1.0 - b2)
    out = []
    for y, signed, d in ((m2, True, words >> 16), (v2.sqrt(), False, words & 0xFFFF)):
        b = _scale_bytes(y)
        s = torch.exp2((127 - b).double()).repeat_interleave(64)[:y.numel()]
        fin = torch.isfinite(y)
        u = (torch.where(fin, y.abs(), 0.0).double() * s * 2.0 ** -120).float().view(torch.int32)
        code = (u + (d << 4 | 8).to(torch.int32)) >> 20
        if not signed:
            code = torch.where((y != 0) & (code == 0), 1, code)
        code = torch.where(fin, code, 0x7F)
        if signed:
            code = code | ((y.view(torch.int32) >> 24) & 0x80)
        out += [code, b]
    return m2, v2, out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip", [False, True])
def test_step8_against_64_bits(dev, dtype, clip):
    """Parameters within the bounds; codes bit for bit those of the fp32 formulas and the
    documented random words, so within one e4m3 step of the exact value."""
    import train_ops

    seed = 0x1234_5678_9ABC_DEF0
    ins = [_inputs(n, n + 1, dtype) for n in SIZES]
    P, G = [i[0].to(dev) for i in ins], [i[1].to(dev) for i in ins]
    st = [_state8(i[2], i[3], dev) for i in ins]
    old = [{k: x.cpu() for k, x in s.items() if k != "step"} for s in st]
    for k, s in enumerate(st):
        s["step"] = 5 * k
    c, scale = 1.0, None
    if clip:
        _, scale = train_ops.grad_norm(G, 1e-6)
        c = float(scale)
    train_ops.adamw_step(P, G, st, 0.01, 0.1, grad_scale=scale, seed=seed)
    for k, (p, g, _, _) in enumerate(ins):
        n, t = SIZES[k], 5 * k + 1
        m, r = _values(old[k]["exp_avg"], old[k]["exp_avg_scale"]), _values(old[k]["exp_rms"], old[k]["exp_rms_scale"])
        want, bound = _exact(p, g, m, r * r, 0.01, 0.1, t, c)
        # r r rounds once more than a stored v: 2 u of d
        up = (want[0] - p.double() * (1 - 0.001)).abs()
        bp = bound[0] + 2 * U * up
        if dtype is torch.bfloat16:
            bp = bp + 2.0 ** -7 * want[0].abs()  # one of the two neighbours: a whole step
        _within(P[k], want[0], bp, f"n={n} p")
        words = _words(n, seed, t, k)
        _, _, (mc, mb, rc, rb) = _plain8(p, g, m.float(), r.float(), 0.01, 0.1, t, words, c)
        s = st[k]
        for got, w in ((s["exp_avg"], mc), (s["exp_avg_scale"], mb), (s["exp_rms"], rc), (s["exp_rms_scale"], rb)):
            assert torch.equal(got.cpu().view(torch.uint8).to(torch.int64).reshape(-1), w.to(torch.int64)), n
        for key, x, b in (("exp_avg", want[1], mb), ("exp_rms", want[2].sqrt(), rb)):
            off = (_values(s[key].cpu(), s[key + "_scale"].cpu()) - x).abs()
            e = bound[1] if key == "exp_avg" else 5 * U * x  # of the fp32 value before rounding
            assert bool((off <= _step_of(x, b) * (1 + 1e-6) + e).all()), (n, key)


@pytest.mark.gpu
def test_step8_rounding_is_unbiased_and_repeats(dev):
    """The mean of (value - exact) / step over N elements: each lies in (-1, 1) with mean 0
    and variance at most 1/4, so six standard deviations are 3 / sqrt(N); 16 random bits
    decide, which leaves a bias of at most 2^-16 steps."""
    import train_ops

    n = 1 << 18
    p, g, m, v = _inputs(n, 5)
    runs = []
    for seed in (1, 1, 2):
        st = _state8(m, v, dev)
        old = {k: x.cpu() for k, x in st.items() if k != "step"}
        st["step"] = 100
        train_ops.adamw_step([p.to(dev)], [g.to(dev)], [st], 0.01, seed=seed)
        runs.append({k: x.cpu().view(torch.uint8) for k, x in st.items() if k != "step"})
    assert all(torch.equal(runs[0][k], runs[1][k]) for k in runs[0])
    assert not torch.equal(runs[0]["exp_avg"], runs[2]["exp_avg"])
    m0, r0 = _values(old["exp_avg"], old["exp_avg_scale"]), _values(old["exp_rms"], old["exp_rms_scale"])
    want, _ = _exact(p, g, m0, r0 * r0, 0.01, 0.0, 101)
    for key, x in (("exp_avg", want[1]), ("exp_rms", want[2].sqrt())):
        step = _step_of(x, runs[0][key + "_scale"])
        err = (_values(runs[0][key].view(torch.float8_e4m3fn), runs[0][key + "_scale"].view(torch.float8_e8m0fnu)) - x) / step
        big = x.abs() > step  # nothing but zero becomes zero among the roots: those are not unbiased
        assert int(big.sum()) > n // 2
        assert abs(float(err[big].mean())) <= 3 / math.sqrt(int(big.sum())) + 2.0 ** -16


@pytest.mark.gpu
def test_step8_moments_fall_without_gradients(dev):
    """What stochastic rounding is for: with zero gradients both moments of every element of
    a block decay although one neighbour keeps the block's scale up."""
    import train_ops

    n = 64 * 512
    m = torch.full((n,), 1e-6)
    v = torch.full((n,), 1e-12)
    p, g = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    g[::64] = 1e-4  # the neighbour
    st = _state8(m, v, dev)
    r0 = float(train_ops.unpack_state8(st["exp_rms"], st["exp_rms_scale"])[1])
    for _ in range(200):
        train_ops.adamw_step([p], [g], [st], 1e-4)
    rest = torch.arange(n, device=dev) % 64 != 0
    m1 = train_ops.unpack_state8(st["exp_avg"], st["exp_avg_scale"])[rest].double()
    r1 = train_ops.unpack_state8(st["exp_rms"], st["exp_rms_scale"])[rest].double()
    # exactly 1e-6 0.9^200 = 7e-16; the lowest code is 2^-30 = 9.3e-10, so of 32256 elements
    # 0.02 are expected not to be zero
    assert float(m1.abs().mean()) < 1e-12
    # 0.999^100 of the root; each of the 32256 elements keeps its expectation, with a standard
    # deviation below 0.3 of it: the mean is known to 6 * 0.3 / sqrt(32256) = 0.01
    assert abs(float(r1.mean()) / r0 - 0.999 ** 100) < 0.01
    assert int((r1 == 0).sum()) == 0


@pytest.mark.gpu
def test_step_zero_gradients_and_zero_state_leave_parameters(dev):
    import train_ops

    for bits in (32, 8):
        p = torch.randn(1000, device=dev)
        before, st = p.clone(), train_ops.adamw_state(p, bits)
        train_ops.adamw_step([p], [torch.zeros_like(p)], [st], 0.1)
        assert torch.equal(p, before)
        assert not any(x.view(torch.uint8).any() for k, x in st.items() if k != "step")


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_step_nonfinite_gradients_stay_with_their_element(dev, bits):
    import train_ops

    n = 640
    p, g, m, v = _inputs(n, 9)
    bad = torch.zeros(n, dtype=torch.bool)
    bad[[0, 70, 77, 639]] = True
    out = []
    for poison in (False, True):
        gg = g.clone()
        gg[bad] = torch.tensor([math.nan, math.inf, -math.inf, math.nan]) if poison else 0.0
        mm, vv = torch.where(bad, 0, m), torch.where(bad, 0, v)  # no part in their blocks' scales
        P = p.clone().to(dev)
        st = {"step": 0, "exp_avg": mm.to(dev), "exp_avg_sq": vv.to(dev)} if bits == 32 else _state8(mm, vv, dev)
        train_ops.adamw_step([P], [gg.to(dev)], [st], 0.01)
        out.append((P.cpu(), {k: x.cpu().view(torch.uint8).view(n, -1) for k, x in st.items()
                              if k != "step" and not k.endswith("scale")}))
    assert torch.equal(out[0][0][~bad], out[1][0][~bad])
    assert torch.isnan(out[1][0][bad]).all()
    for k in out[0][1]:
        assert torch.equal(out[0][1][k][~bad], out[1][1][k][~bad]), k
    if bits == 8:
        assert bool(((out[1][1]["exp_avg"][bad] & 0x7F) == 0x7F).all()) and bool((out[1][1]["exp_rms"][bad] == 0x7F).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_step_views_of_flat_buffers_at_any_offset(dev, dtype, bits):
    """Tensors that start at odd elements of flat buffers, 90 of them with empty ones (three
    launches), next to a second width in the same list: as separate tensors, and nothing
    between the views is written."""
    import train_ops

    sizes = [(k * 37) % 130 for k in range(88)] + [5000, 3333]
    offs, at = [], 1
    for n in sizes:
        offs.append(at)
        at += n + 1 + n % 3

    def views(x):
        return [x[o:o + n] for o, n in zip(offs, sizes)]

    p, g, m, v = _inputs(at, 3, dtype)
    flat = {"p": p.to(dev), "g": g.to(dev)}
    keep = flat["p"].clone()
    if bits == 32:
        flat["exp_avg"], flat["exp_avg_sq"] = m.to(dev), v.to(dev)
        st = [{"step": 1, "exp_avg": a, "exp_avg_sq": b} for a, b in zip(views(flat["exp_avg"]), views(flat["exp_avg_sq"]))]
    else:
        whole = _state8(m, v, dev)
        flat["exp_avg"], flat["exp_rms"] = whole["exp_avg"], whole["exp_rms"]
        st = []
        for a, b in zip(views(whole["exp_avg"]), views(whole["exp_rms"])):
            nb = -(-a.numel() // 64)
            sc = torch.full((2, nb), 110, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)
            st.append({"step": 1, "exp_avg": a, "exp_avg_scale": sc[0], "exp_rms": b, "exp_rms_scale": sc[1]})
    states = {k: flat[k].clone() for k in flat if k.startswith("exp")}
    alone = [{k: (x.clone() if k != "step" else x) for k, x in s.items()} for s in st]
    pa = [x.clone() for x in views(flat["p"])]
    train_ops.adamw_step(views(flat["p"]), views(flat["g"]), st, 0.01, 0.1, seed=7)
    train_ops.adamw_step(pa, [x.clone() for x in views(flat["g"])], alone, 0.01, 0.1, seed=7)
    inside = torch.zeros(at, dtype=torch.bool, device=dev)
    for x in views(inside):
        x.fill_(True)
    raw = lambda x: x.view(torch.uint8).view(at, -1)  # noqa: E731
    assert torch.equal(raw(flat["p"])[~inside], raw(keep)[~inside])
    for k, x in states.items():
        assert torch.equal(raw(flat[k])[~inside], raw(x)[~inside]), k
    for a, b in zip(views(flat["p"]), pa):
        assert torch.equal(a, b)
    for s, q in zip(st, alone):
        for k in s:
            assert s[k] == q[k] if k == "step" else torch.equal(s[k].view(torch.uint8), q[k].view(torch.uint8)), k


@pytest.mark.gpu
def test_step_mixes_widths_and_dtypes_in_one_list(dev):
    import train_ops

    kinds = [(torch.float32, 32), (torch.bfloat16, 8), (torch.float32, 8), (torch.bfloat16, 32)] * 2
    ps, gs, st = [], [], []
    for k, (dt, bits) in enumerate(kinds):
        p, g, m, v = _inputs(500 + k, k, dt)
        ps.append(p.to(dev)), gs.append(g.to(dev))
        st.append(_state8(m, v, dev) if bits == 8 else {"step": 0, "exp_avg": m.to(dev), "exp_avg_sq": v.to(dev)})
    one_p = [p.clone() for p in ps]
    one_s = [{k: (x.clone() if k != "step" else x) for k, x in s.items()} for s in st]
    train_ops.adamw_step(ps, gs, st, 0.01, seed=3)
    from diff_gaussian_rasterization import _C

    lib = _C.load_library()
    for k, (dt, bits) in enumerate(kinds):  # each by itself, at its own place in the list
        s = one_s[k]
        second = s["exp_avg_sq"] if bits == 32 else s["exp_rms"]
        seg = _C.GsrAdamWSegment(one_p[k].data_ptr(), gs[k].data_ptr(), s["exp_avg"].data_ptr(), second.data_ptr(),
                                 None if bits == 32 else s["exp_avg_scale"].data_ptr(),
                                 None if bits == 32 else s["exp_rms_scale"].data_ptr(), 500 + k, 0.01, 0.0, 1, k)
        _C._check(lib.gsr_adamw_step(ctypes.byref(seg), 1, _C.DTYPES[dt], bits, 0.9, 0.999, 1e-15, None, 3,
                                     _C._stream(dev)), "gsr_adamw_step")
        assert torch.equal(one_p[k], ps[k])
        for key in s:
            if key != "step":
                assert torch.equal(s[key].view(torch.uint8), st[k][key].view(torch.uint8)), (k, key)


@pytest.mark.gpu
def test_step_refusals_leave_everything_as_it_was(dev):
    import train_ops

    p, g = torch.randn(8, 4, device=dev), torch.randn(8, 4, device=dev)
    st = train_ops.adamw_state(p, 8)
    cases = [
        (dict(grads=[g, g.half()]), "dtype"), (dict(params=[p, p]), "twice"), (dict(params=[p, p.t()]), "parameter"),
        (dict(grads=[g, g[:4]]), "gradient"), (dict(grads=[g, g.t().contiguous().t()]), "contiguous"),
        (dict(params=[p, p.cpu()]), "GPU"), (dict(grads=[g, g.cpu()]), "expected cuda"),
        (dict(states=[st, {**st, "exp_rms": st["exp_avg_scale"]}]), "exp_rms"),
        (dict(states=[st, {"step": 0, "exp_avg": p}]), "exp_avg"),
        (dict(states=[st, {**st, "exp_avg_scale": st["exp_avg_scale"][:0]}]), "exp_avg_scale"),
        (dict(grad_scale=torch.ones(2, device=dev)), "grad_scale"), (dict(grad_scale=torch.ones(())), "grad_scale"),
        (dict(betas=(0.9, 1.0)), "betas"), (dict(eps=-1.0), "eps"),
        (dict(states=[st, st]), "twice"),
    ]
    q = torch.randn(8, 4, device=dev)
    for kw, msg in cases:
        before = (p.clone(), q.clone())
        args = dict(params=[p, q], grads=[g, g.clone()], states=[st, train_ops.adamw_state(q, 8)], lr=0.1)
        args.update(kw)
        with pytest.raises(RuntimeError, match=msg):
            train_ops.adamw_step(**args)
        assert torch.equal(p, before[0]) and torch.equal(q, before[1]) and st["step"] == 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x = g * 2  # something to capture
        with pytest.raises(RuntimeError, match="capture"):
            train_ops.adamw_step([p], [g], [st], 0.1)
    assert st["step"] == 0 and x is not None


@pytest.mark.gpu
def test_step_raises_for_a_graph_that_saved_the_parameter(dev):
    import train_ops

    p = torch.randn(10, device=dev, requires_grad=True)
    y = (p * p).sum()
    train_ops.adamw_step([p], [torch.ones(10, device=dev)], [train_ops.adamw_state(p)], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
def test_step_a_bad_count_in_one_launch_stops_all(dev):
    import struct

    import train_ops

    ps = [torch.ones(5, device=dev), torch.ones(5, device=dev)]
    st = [train_ops.adamw_state(ps[0]), train_ops.adamw_state(ps[1], 8)]
    st[1]["step"] = 2 ** 31 - 1
    with pytest.raises(struct.error):
        train_ops.adamw_step(ps, [p.clone() for p in ps], st, 0.1)
    assert st[0]["step"] == 0 and all(torch.equal(p, torch.ones_like(p)) for p in ps)


@pytest.mark.gpu
def test_step_takes_numpy_rates_and_inference_tensors(dev):
    import train_ops

    with torch.inference_mode():
        p = torch.ones(5, device=dev)
        train_ops.adamw_step([p], [torch.ones(5, device=dev)], [train_ops.adamw_state(p)], np.float32(0.5),
                             weight_decay=np.float64(0.0))
        # the first step is lr g / |g|, to 2^-23 of its roundings
        np.testing.assert_allclose(p.cpu().numpy(), 0.5, rtol=1e-5)


@pytest.mark.gpu
def test_step_on_another_stream(dev):
    import train_ops

    p, g, m, v = (x.to(dev) for x in _inputs(100_003, 1))
    ref = p.clone()
    train_ops.adamw_step([ref], [g], [{"step": 0, "exp_avg": m.clone(), "exp_avg_sq": v.clone()}], 0.01)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm, scale = train_ops.grad_norm([g])
        train_ops.adamw_step([p], [g], [{"step": 0, "exp_avg": m, "exp_avg_sq": v}], 0.01, grad_scale=scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(p, ref)


@pytest.mark.gpu
def test_step8_beyond_32_bit_offsets(dev):
    """2^32 + 200 elements in bf16: the last elements and their scales are reached, by the
    random words of their own 64-bit index."""
    import train_ops

    n, tail = (1 << 32) + 200, 264
    p = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    tp, tg, _, _ = _inputs(tail, 2, torch.bfloat16)
    p[-tail:], g[-tail:] = tp.to(dev), tg.to(dev)
    st = train_ops.adamw_state(p, 8)
    norm, scale = train_ops.grad_norm([g])
    want = float(tg.double().norm())
    assert abs(float(norm) - want) <= 2 * U * want
    train_ops.adamw_step([p], [g], [st], 0.01, seed=5)
    z = torch.zeros(tail)
    i = torch.arange(n - tail, n, dtype=torch.int64)
    key = _mix((_mix((_mix((_mix(5) + 0) & M32) + 1) & M32) + 0) & M32)
    words = _mix(((i & M32) * 0x9E3779B9 + (i >> 32) * 0x3C6EF373 + key) & M32)
    assert (n - tail) % 64 == 0  # the tail's blocks are its own
    _, _, (mc, mb, rc, rb) = _plain8(tp, tg, z, z, 0.01, 0.0, 1, words)
    for k, w in (("exp_avg", mc), ("exp_rms", rc), ("exp_avg_scale", mb), ("exp_rms_scale", rb)):
        got = st[k][-w.numel():].cpu().view(torch.uint8)
        assert torch.equal(got.long(), w.long()), k
    want, bound = _exact(tp, tg, z, z, 0.01, 0.0, 1)
    _within(p[-tail:], want[0], bound[0] + 2.0 ** -7 * want[0].abs() + 2 * U * 0.01, "p")
    assert not p[:-tail].any()


# ------------------------------------------------------------------ GPU: the norm
@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [3], [4096], [4097], [0, 5, 0], [100_003, 1, 4095, 12_288],
                                   [k % 97 for k in range(300)], [20_000_000]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_grad_norm_against_64_bits(dev, sizes, dtype):
    import train_ops

    flat = torch.randn(sum(sizes) + 1, device=dev).to(dtype)
    gs = list(flat[1:].split(sizes))  # at odd elements
    want = float(flat[1:].double().norm())
    norm, scale = train_ops.grad_norm(gs, 0.5)
    assert abs(float(norm) - want) <= 2 * U * want
    c = min(1.0, 0.5 / (want + 1e-6))
    assert abs(float(scale) - c) <= 2 * U * c
    norm, scale = train_ops.grad_norm(gs)
    assert float(scale) == 1.0


@pytest.mark.gpu
def test_grad_norm_extremes(dev):
    import train_ops

    f = lambda *x: [float(v) for v in train_ops.grad_norm([torch.tensor(x, device=dev)], 1.0)]  # noqa: E731
    assert f(0.0, 0.0) == [0.0, 1.0]
    norm, scale = f(1e30, -1e30)  # the squares pass fp32's range
    assert abs(norm / (1e30 * math.sqrt(2)) - 1) < 4 * U and abs(scale * norm - 1) < 4 * U
    norm, scale = f(1e-30, 1e-30)
    assert abs(norm / (1e-30 * math.sqrt(2)) - 1) < 4 * U and scale == 1.0
    assert f(math.inf, 1.0) == [math.inf, 0.0]
    norm, scale = f(math.nan, 1.0)
    assert math.isnan(norm) and math.isnan(scale)
    a, b = torch.randn(1000, device=dev), torch.randn(50, device=dev).bfloat16()  # dtypes side by side
    want = math.hypot(float(a.double().norm()), float(b.double().norm()))
    assert abs(float(train_ops.grad_norm([a, b])[0]) - want) <= 2 * U * want


@pytest.mark.gpu
def test_grad_norm_captured_and_replayed(dev):
    import train_ops

    gs = [torch.randn(100_000, device=dev), torch.randn(77, device=dev)]
    train_ops.grad_norm(gs, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, scale = train_ops.grad_norm(gs, 1.0)
    for k in range(4):
        gs[0].mul_(1.5).add_(k)
        eager = train_ops.grad_norm(gs, 1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager[0]) and torch.equal(scale, eager[1])


@pytest.mark.gpu
def test_train_state_runs_with_8_bit_states(dev):
    """The model's own training step on 8-bit states, clipped and decayed, beside the 32-bit one:
    the first step's parameters agree (both start from zero moments, which 8 bits hold), and
    it keeps running."""
    import synthetic
    import train_step

    cam = synthetic.make_camera(128, 96, 0).to(dev)
    target = synthetic.make_target(128, 96, seed=1).to(dev)
    bg = torch.zeros(3, device=dev)
    got = {}
    for bits in (32, 8):
        g = synthetic.make_gaussians(3000, 2, seed=0).to(dev, requires_grad=True)
        st = train_step.TrainState(g, spatial_lr_scale=1.0, fused=True, state_bits=bits, weight_decay=0.01, max_norm=1e-3)
        train_step.full_train_step(1, cam, g, st, target, bg)
        got[bits] = ([p.detach().clone() for p in g.params()], st.optimizer.grad_norm.clone())
        for it in (2, 3, 4):
            loss = train_step.full_train_step(it, cam, g, st, target, bg)
        assert torch.isfinite(loss) and all(torch.isfinite(p).all() for p in g.params())
        assert all(s["step"] == 4 for s in st.optimizer.state.values())
    lrs = [0.00016, 0.0025, 0.0025 / 20, 0.05, 0.005, 0.001]
    for a, b, lr in zip(got[32][0], got[8][0], lrs):
        # the two renders' gradients differ by the order of atomics; Adam's first step is
        # lr g / |g|, so an entry whose gradient is lost in that noise may flip
        d = (a - b).abs()
        assert float((d > 1e-3 * lr + 4 * U * a.abs()).float().mean()) < 1e-2
        assert float(d.max()) <= 2 * lr + 1e-6
    np.testing.assert_allclose(float(got[32][1]), float(got[8][1]), rtol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(dev, bits, tmp_path):
    """Saved, loaded with the safe loader into another optimiser, and continued: the same bits."""
    import train_ops

    gen = torch.Generator().manual_seed(0)
    base = [torch.randn(77, 3, generator=gen), torch.randn(5, generator=gen), torch.randn(0, 3)]
    grads = [[torch.randn(b.shape, generator=gen).to(dev) for b in base] for _ in range(4)]

    def make():
        ps = [b.clone().to(dev).requires_grad_(True) for b in base]
        return ps, train_ops.FusedAdamW([{"params": ps[:2], "lr": 0.1, "name": "a"}, {"params": ps[2:]}],
                                        state_bits=bits, weight_decay=0.1, max_norm=1.0, seed=5)

    def run(ps, opt, steps):
        for k in steps:
            for p, g in zip(ps, grads[k]):
                p.grad = g
            opt.step()

    pa, oa = make()
    run(pa, oa, range(2))
    path = tmp_path / "opt.pt"
    torch.save(oa.state_dict(), path)
    pb, ob = make()
    for p, q in zip(pa, pb):
        q.data.copy_(p.data)
    ob.param_groups[0]["lr"] = 0.5
    ob.load_state_dict(torch.load(path, weights_only=True))
    assert ob.param_groups[0]["lr"] == 0.1 and ob.param_groups[0]["name"] == "a"
    run(pa, oa, range(2, 4))
    run(pb, ob, range(2, 4))
    for p, q in zip(pa, pb):
        assert torch.equal(p, q) and oa.state[p]["step"] == ob.state[q]["step"] == 4
    with pytest.raises(ValueError, match="param groups"):
        ob.load_state_dict({"state": {}, "param_groups": []})
    bad = oa.state_dict()
    bad["state"][0]["exp_avg"] = bad["state"][0]["exp_avg"][:5]
    with pytest.raises(RuntimeError, match="exp_avg"):
        ob.load_state_dict(bad)


# ------------------------------------------------------------------ GPU: values that are not their bytes
def _negated(x):
    """x as a view of -x's bytes, as the backward of a conjugated complex number leaves it."""
    return torch._neg_view(-x)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_step_takes_negated_gradients_and_scale(dev, bits):
    import train_ops

    for n in (1, 777):
        p, g, m, v = _inputs(n, n + 3)
        assert g.any()
        got = []
        for neg_grad, neg_scale in ((False, False), (True, False), (False, True)):
            P, G, scale = p.to(dev), g.to(dev), torch.tensor(0.25, device=dev)
            G, scale = _negated(G) if neg_grad else G, _negated(scale) if neg_scale else scale
            assert G.is_contiguous() and G.is_neg() == neg_grad and scale.is_neg() == neg_scale
            st = {"step": 3, "exp_avg": m.to(dev), "exp_avg_sq": v.to(dev)} if bits == 32 else _state8(m, v, dev)
            train_ops.adamw_step([P], [G], [st], 0.01, grad_scale=scale)
            got.append([P] + [x.view(torch.uint8) for k, x in st.items() if k != "step"])
        for other in got[1:]:
            assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.gpu
def test_optimiser_takes_the_gradient_that_a_complex_loss_leaves(dev):
    """b.grad of one element is contiguous and a negated view."""
    import train_ops

    def loss(a, b):
        return (torch.complex(a, b).conj() * torch.tensor([0.3 - 0.7j], device=dev)).real.sum()

    new = lambda: [torch.ones(1, device=dev, requires_grad=True) for _ in range(2)]  # noqa: E731
    pa, pb = new(), new()
    opt = train_ops.FusedAdamW([{"params": pa, "lr": 0.1}], eps=1e-8, max_norm=1.0)
    ref = torch.optim.AdamW(pb, lr=0.1, eps=1e-8, weight_decay=0.0)
    for _ in range(3):
        loss(*pa).backward()
        loss(*pb).backward()
        assert pa[1].grad.is_neg() and pa[1].grad.is_contiguous()
        for q in pb:
            q.grad = q.grad.resolve_neg()  # torch's list operations refuse it
        opt.step()
        torch.nn.utils.clip_grad_norm_(pb, 1.0)
        ref.step()
        opt.zero_grad()
        ref.zero_grad()
    # three steps of about 14 roundings each, of values of order 1
    torch.testing.assert_close(torch.cat(pa), torch.cat(pb), rtol=0, atol=3 * 14 * U)


@pytest.mark.gpu
def test_step_refuses_negated_parameters_and_states(dev):
    import train_ops

    p, g = torch.randn(6, device=dev), torch.randn(6, device=dev)
    for kw, msg in ((dict(params=[_negated(p)]), "negated"), (dict(key="exp_avg"), "exp_avg"),
                    (dict(key="exp_avg_sq"), "exp_avg_sq")):
        st = train_ops.adamw_state(p)
        if "key" in kw:
            st[kw["key"]] = _negated(st[kw["key"]])
        q = kw.get("params", [p])
        before = q[0].clone()
        with pytest.raises(RuntimeError, match=msg):
            train_ops.adamw_step(q, [g], [st], 0.1)
        assert torch.equal(q[0], before) and st["step"] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["negative", "missing", "large"])
def test_step_a_refusal_of_a_later_kind_comes_before_the_first_launch(dev, what):
    """Lists whose tensors go out in several launches: what the second would refuse stops all."""
    import train_ops

    p, q = torch.ones(5, device=dev), torch.ones(5, device=dev)
    states = [train_ops.adamw_state(p), train_ops.adamw_state(q, 8)]
    grads = [torch.ones_like(p), torch.ones_like(q)]
    if what == "negative":
        states[1]["step"] = -1
    elif what == "missing":  # of an empty tensor, which goes out in no launch
        q, grads[1] = q[:0], grads[1][:0]
        states[1] = train_ops.adamw_state(q, 8)
        del states[1]["step"]
    else:  # never touched: the gradient is the parameter itself
        q = torch.empty((1 << 33) + 1, dtype=torch.bfloat16, device=dev)
        grads[1] = q
        codes = lambda: torch.empty(q.numel(), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)  # noqa: E731
        scale = lambda: torch.empty((1 << 27) + 1, dtype=torch.uint8, device=dev).view(torch.float8_e8m0fnu)  # noqa: E731
        states[1] = {"step": 0, "exp_avg": codes(), "exp_rms": codes(), "exp_avg_scale": scale(), "exp_rms_scale": scale()}
    count = states[1].get("step")
    with pytest.raises(RuntimeError, match="size" if what == "large" else "step"):
        train_ops.adamw_step([p, q], grads, states, 0.1)
    assert torch.equal(p, torch.ones_like(p)) and not states[0]["exp_avg"].any() and not states[0]["exp_avg_sq"].any()
    assert states[0]["step"] == 0 and states[1].get("step") == count


@pytest.mark.gpu
def test_step_refuses_states_that_share_any_buffer(dev):
    """Every buffer that the step writes: a shared one would be read and written by two workgroups at once."""
    import train_ops

    ps = [torch.ones(100, device=dev), torch.ones(100, device=dev)]
    gs = [torch.ones(100, device=dev)] * 2  # gradients are only read
    for bits, keys in ((32, ("exp_avg", "exp_avg_sq")), (8, ("exp_avg", "exp_avg_scale", "exp_rms", "exp_rms_scale"))):
        for key in keys:
            st = [train_ops.adamw_state(p, bits) for p in ps]
            st[1][key] = st[0][key]
            with pytest.raises(RuntimeError, match="twice"):
                train_ops.adamw_step(ps, gs, st, 0.1)
            assert st[0]["step"] == st[1]["step"] == 0
        one = train_ops.adamw_state(ps[0], bits)
        one[keys[-1]] = one[keys[-1] if bits == 32 else "exp_avg_scale"]
        if bits == 32:
            one["exp_avg_sq"] = one["exp_avg"]
        with pytest.raises(RuntimeError, match="twice"):
            train_ops.adamw_step(ps[:1], gs[:1], [one], 0.1)
    st = train_ops.adamw_state(ps[0])
    with pytest.raises(RuntimeError, match="twice"):  # a state that is another tensor's parameter
        train_ops.adamw_step(ps, gs, [{**st, "exp_avg_sq": ps[1]}, train_ops.adamw_state(ps[1])], 0.1)
    assert all(torch.equal(p, torch.ones_like(p)) for p in ps)
    train_ops.adamw_step(ps, gs, [train_ops.adamw_state(p) for p in ps], 0.1)  # a shared gradient is in order
    assert torch.equal(ps[0], ps[1])


def _adamw_on_cpu(**kw):
    import train_ops

    ps = [torch.ones(3, requires_grad=True), torch.ones(2, requires_grad=True)]
    return ps, train_ops.FusedAdamW([{"params": ps[:1], "lr": 0.1}, {"params": ps[1:]}], **kw)


def test_load_state_dict_takes_the_hyperparameters_of_a_torch_checkpoint():
    _, opt = _adamw_on_cpu(seed=4, max_norm=2.0)
    qs = [torch.ones(3, requires_grad=True), torch.ones(2, requires_grad=True)]
    ref = torch.optim.AdamW([{"params": qs[:1]}, {"params": qs[1:]}], lr=0.3, betas=(0.5, 0.6), eps=1e-8)
    for q in qs:
        q.grad = torch.ones_like(q)
    ref.step()
    opt.load_state_dict(ref.state_dict())
    assert opt.betas == (0.5, 0.6) and opt.eps == 1e-8
    assert opt.param_groups[0]["lr"] == 0.3 and opt.param_groups[0]["weight_decay"] == 0.01
    assert opt.seed == 4 and opt.max_norm == 2.0  # not in such a checkpoint: as constructed
    assert all(s["step"] == 1 for s in opt.state.values()) and len(opt.state) == 2


def test_state_dict_holds_all_that_a_step_depends_on():
    ps, a = _adamw_on_cpu(betas=(0.8, 0.9), eps=1e-6, seed=7, max_norm=3.0, state_bits=8, weight_decay=0.1)
    _, b = _adamw_on_cpu()
    b.load_state_dict(a.state_dict())
    assert (b.betas, b.eps, b.seed, b.max_norm, b.state_bits) == ((0.8, 0.9), 1e-6, 7, 3.0, 8)
    assert [g["weight_decay"] for g in b.param_groups] == [0.1, 0.1]
    # torch's own optimiser takes it too
    ref = torch.optim.AdamW([{"params": ps[:1]}, {"params": ps[1:]}], lr=0.3)
    ref.load_state_dict(a.state_dict())
    assert ref.param_groups[0]["betas"] == (0.8, 0.9) and ref.param_groups[0]["eps"] == 1e-6
    b.betas, b.eps = (0.7, 0.95), 1e-9
    assert all(g["betas"] == (0.7, 0.95) and g["eps"] == 1e-9 for g in b.param_groups)


def test_a_group_without_betas_goes_by_the_optimisers():
    import train_ops

    _, opt = _adamw_on_cpu(betas=(0.8, 0.9))
    opt.param_groups.append({"params": [torch.ones(1)], "lr": 0.1, "weight_decay": 0.0})
    assert opt.betas == (0.8, 0.9) and opt.eps == 1e-15
    opt.betas = (0.5, 0.6)
    assert opt.betas == (0.5, 0.6) and train_ops.FusedAdamW([], eps=1e-3).eps == 1e-3


@pytest.mark.parametrize("change, msg", [(dict(amsgrad=True), "amsgrad"), (dict(maximize=True), "maximize"),
                                         (dict(betas=(0.5, 0.9)), "betas"), (dict(eps=1e-3), "eps"),
                                         (dict(decoupled_weight_decay=False, weight_decay=0.1), "decoupled")])
def test_options_that_a_step_would_ignore_are_refused(change, msg):
    import train_ops

    ps, opt = _adamw_on_cpu()
    with pytest.raises(ValueError, match=msg):  # at construction
        train_ops.FusedAdamW([{"params": ps[:1]}, {"params": ps[1:], **change}])
    d = opt.state_dict()
    d["param_groups"][1].update(change)
    d["param_groups"][0]["lr"] = 9.0
    d["seed"] = 5
    d["state"] = {0: {**train_ops.adamw_state(ps[0]), "step": 3}}
    with pytest.raises(ValueError, match=msg):  # on loading, which then changes nothing
        opt.load_state_dict(d)
    assert opt.param_groups[0]["lr"] == 0.1 and opt.seed == 0 and not opt.state
    opt.param_groups[1].update(change)
    for p in ps:
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError, match=msg):  # and at the step
        opt.step()


@pytest.mark.gpu
def test_step_after_loading_goes_by_the_checkpoints_betas_and_eps(dev):
    """A torch.optim.AdamW checkpoint with its own betas and eps, continued by both."""
    import train_ops

    gen = torch.Generator().manual_seed(3)
    base, grads = torch.randn(500, generator=gen), [torch.randn(500, generator=gen).to(dev) for _ in range(4)]
    q = base.clone().to(dev).requires_grad_(True)
    ref = torch.optim.AdamW([q], lr=0.01, betas=(0.5, 0.6), eps=1e-3, weight_decay=0.0)
    for g in grads[:2]:
        q.grad = g
        ref.step()
    p = q.detach().clone().requires_grad_(True)
    opt = train_ops.FusedAdamW([{"params": [p]}])
    opt.load_state_dict(ref.state_dict())
    for g in grads[2:]:
        p.grad = q.grad = g
        opt.step()
        ref.step()
    # two steps: 3 roundings of p each and 12 of updates of at most about 2 lr; moments of order 1
    torch.testing.assert_close(p, q, rtol=8 * U, atol=2 * 12 * U * 0.02 + 8 * U * 0.02)
    torch.testing.assert_close(opt.state[p]["exp_avg_sq"], ref.state[q]["exp_avg_sq"], rtol=12 * U, atol=0)


def test_train_state_adamw_options():
    import synthetic
    import train_ops
    import train_step

    g = synthetic.make_gaussians(4, 1)
    with pytest.raises(ValueError, match="state_bits"):
        train_step.TrainState(g, 1.0, fused=True, state_bits=0)
    opt = train_step.TrainState(g, 1.0, fused=True, state_bits=8, seed=11).optimizer
    assert isinstance(opt, train_ops.FusedAdamW) and opt.seed == 11 and opt.state_bits == 8
    assert train_step.TrainState(g, 1.0, fused=True, max_norm=1.0).optimizer.state_bits == 32
    for fused in (False, True):
        with pytest.raises(ValueError, match="seed"):  # of nothing that would use it
            train_step.TrainState(g, 1.0, fused=fused, seed=11)


def test_train_state_decays_the_groups_that_are_named():
    import synthetic
    import train_step

    g = synthetic.make_gaussians(4, 1)
    decay = lambda wd: [x["weight_decay"] for x in  # noqa: E731
                        train_step.TrainState(g, 1.0, fused=True, weight_decay=wd).optimizer.param_groups]
    assert decay(0.1) == [0.1] * 6
    assert decay({"f_rest": 0.1, "opacity": 0.2}) == [0.0, 0.0, 0.1, 0.2, 0.0, 0.0]
    with pytest.raises(ValueError, match="positions"):
        train_step.TrainState(g, 1.0, fused=True, weight_decay={"positions": 0.1})
    with pytest.raises(ValueError, match="fused"):
        train_step.TrainState(g, 1.0, weight_decay={"f_rest": 0.1})


# ------------------------------------------------------------------ GPU: bit for bit
RCP = {32: False, 8: True}  # whose quotient is a product with the hardware's reciprocal


def _fp32_step(p, g, m, v, lr, wd, t, c=1.0, rcp=False, betas=(0.9, 0.999), eps=1e-15):
    """(all the values that p' may have, m', v') by the formulas in numpy's fp32, where each operation
    rounds once (torch's square root on the CPU does not round to nearest).  ``rcp``: the quotient
    is a product with a reciprocal that is off by one ulp at most, so its value to nearest or one
    of the two numbers next to it; else it rounds once itself."""
    f, (b1, b2) = np.float32, betas
    p, g, m, v = (x.float().numpy() for x in (p, g, m, v))
    x = g * f(c)
    m2, v2 = m + (x - m) * f(1 - b1), v * f(b2) + (x * x) * f(1 - b2)
    d = np.sqrt(v2) * f(1 / math.sqrt(1 - b2 ** t)) + f(eps)
    if rcp:
        r = f(1) / d
        quotients = [m2 * y for y in (r, np.nextafter(r, f(0)), np.nextafter(r, f(np.inf)))]
    else:
        quotients = [m2 / d]
    ps = [p * f(1 - lr * wd) + q * f(-lr / (1 - b1 ** t)) for q in quotients]
    assert all(y.dtype == f for y in ps + [m2, v2])
    return [torch.from_numpy(y) for y in ps], torch.from_numpy(m2), torch.from_numpy(v2)


def _dithered(p2, words):
    """Rounded to bf16 by 16 bits formed of the element's word: up where the dropped bits and they carry."""
    low = (((words * 0x9E3779B9) & M32) >> 16).to(torch.int32)
    return ((p2.view(torch.int32) + low) & -0x10000).view(torch.float32).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_step_bit_for_bit(dev, dtype, clip, bits):
    """Parameters and 32-bit moments are those of the formulas in fp32, each operation rounded by
    itself; a bf16 parameter is rounded by the documented random bits."""
    import train_ops

    seed, sizes = 0xFEDC_BA98_7654_3210, SIZES + [100_003]
    ins = [_inputs(n, n + 2, dtype) for n in sizes]
    P, G = [i[0].to(dev) for i in ins], [i[1].to(dev) for i in ins]
    st = [_state8(i[2], i[3], dev) if bits == 8 else {"exp_avg": i[2].to(dev), "exp_avg_sq": i[3].to(dev)} for i in ins]
    old = [{k: x.cpu() for k, x in s.items() if k != "step"} for s in st]
    for k, s in enumerate(st):
        s["step"] = 7 * k
    c, scale = 1.0, None
    if clip:
        _, scale = train_ops.grad_norm(G, 1e-6)
        c = float(scale)
    train_ops.adamw_step(P, G, st, 0.01, 0.1, grad_scale=scale, seed=seed)
    for k, (p, g, m, v) in enumerate(ins):
        n, t = sizes[k], 7 * k + 1
        words = _words(n, seed, t, k)
        if bits == 8:
            m = _values(old[k]["exp_avg"], old[k]["exp_avg_scale"]).float()
            r = _values(old[k]["exp_rms"], old[k]["exp_rms_scale"]).float()
            v = r * r
        want, m2, v2 = _fp32_step(p, g, m, v, 0.01, 0.1, t, c, rcp=RCP[bits])
        if bits == 32:
            assert torch.equal(st[k]["exp_avg"].cpu(), m2) and torch.equal(st[k]["exp_avg_sq"].cpu(), v2), n
        if dtype is torch.bfloat16:
            want = [_dithered(w, words) for w in want]
        hit = torch.stack([P[k].cpu() == w for w in want]).any(0)
        assert bool(hit.all()), (n, int((~hit).sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_bf16_rounding_is_unbiased(dev, bits):
    """(rounded - exact) / step over N elements lies in (-1, 1) with mean 0 and variance at most
    1/4: six standard deviations are 3 / sqrt(N); every one of the 2^16 dropped patterns has
    its own share of the 2^16 random ones, so there is no bias but the fp32 value's own error, far
    below 2^-10 of a step."""
    import train_ops

    n = 1 << 18
    p, g, m, v = _inputs(n, 11, torch.bfloat16)
    st = {"step": 50, "exp_avg": m.to(dev), "exp_avg_sq": v.to(dev)} if bits == 32 else {**_state8(m, v, dev), "step": 50}
    if bits == 8:
        m = _values(st["exp_avg"].cpu(), st["exp_avg_scale"].cpu())
        v = _values(st["exp_rms"].cpu(), st["exp_rms_scale"].cpu()) ** 2
    P = p.to(dev)
    train_ops.adamw_step([P], [g.to(dev)], [st], 0.01, 0.1, seed=3)
    want = _exact(p, g, m, v, 0.01, 0.1, 51)[0][0]
    step = torch.exp2(torch.frexp(want)[1].double() - 8)
    err = (P.cpu().double() - want) / step
    assert float(err.abs().max()) < 1 + 2.0 ** -10
    assert float((err != 0).float().mean()) > 0.9
    assert abs(float(err.mean())) <= 3 / math.sqrt(n) + 2.0 ** -10


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_bf16_parameters_follow_updates_far_below_half_a_step(dev, bits):
    """From zero moments the first update is lr g / |g|.  Of 1.5 (steps of 2^-7) an lr of 2^-13
    moves one element in 64 by a whole step: the mean of N moves by 2^-13, with a standard deviation
    of 2^-7 sqrt(63) / 64 / sqrt(N) < 2^-19; rounded to nearest none would move."""
    import train_ops

    n = 1 << 18
    p = torch.full((n,), 1.5, dtype=torch.bfloat16, device=dev)
    g = torch.full((n,), 1e-3, dtype=torch.bfloat16, device=dev)
    train_ops.adamw_step([p], [g], [train_ops.adamw_state(p, bits)], 2.0 ** -13, seed=9)
    assert set(p.unique().tolist()) == {1.5, 1.5 - 2.0 ** -7}
    # the update itself: 14 u of 2^-13
    assert abs(1.5 - float(p.double().mean()) - 2.0 ** -13) <= 6 * 2.0 ** -19 + 14 * U * 2.0 ** -13


@pytest.mark.gpu
def test_grad_norm_infinite_norm_and_bound(dev):
    """As torch's clipping: an infinite norm over an infinite bound is NaN; a finite one is not scaled."""
    import train_ops

    g = torch.tensor([1.0, math.inf], device=dev)
    norm, scale = train_ops.grad_norm([g], math.inf)
    assert math.isinf(float(norm)) and math.isnan(float(scale))
    assert float(train_ops.grad_norm([g[:1]], math.inf)[1]) == 1.0
    p = torch.ones(2, device=dev, requires_grad=True)
    p.grad = g.clone()
    torch.nn.utils.clip_grad_norm_([p], math.inf)
    assert bool(torch.isnan(p.grad).all())
