"""Eviction to a budget: selection by an accumulated weight and the gathered rows of many
tensors, 8-bit optimiser states among them.  Selections and plain rows are exact; 8-bit rows
are compared bit for bit with their definition in 64 bits (powers of two and 4-bit
significands: every operation before the one rounding is exact)."""
import ctypes
import math

import pytest
import torch


# ------------------------------------------------------------------ plain forms
def _select(score, budget, protect=None):
    """Sorted by (protected, a number, value) from the top, stable: of equals the lowest index."""
    score = score.reshape(-1).tolist()
    flags = [False] * len(score) if protect is None else protect.tolist()

    def key(i):
        if flags[i]:
            return (0, 0, 0.0)  # all protected rows are alike
        return (1, 1, 0.0) if math.isnan(score[i]) else (1, 0, -score[i])

    return sorted(sorted(range(len(score)), key=key)[:budget])


def _values(codes, scale):
    b = scale.view(torch.uint8).double()
    return (codes.reshape(-1).double() * torch.exp2(b - 127).repeat_interleave(64)[:codes.numel()]).view(codes.shape)


def _encode(x, signed):
    """e4m3 codes and scale bytes of x (64 bits) by comparison with all the code values:
    the nearest, ties to the even code; without sign nothing but zero becomes zero."""
    n = x.numel()
    x = x.reshape(-1)
    fin = torch.isfinite(x)
    a = torch.where(fin, x.abs(), 0.0)
    full = torch.nn.functional.pad(a, (0, -n % 64)).view(-1, 64).amax(1)
    e = torch.frexp(full)[1] - 1
    byte = torch.where(full > 0, (e - 7 + 127).clamp_min(0), 0)
    t = a / torch.exp2(byte.double() - 127).repeat_interleave(64)[:n]
    table = torch.arange(0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    hi = torch.searchsorted(table, t).clamp(1, 0x7E)
    lo = hi - 1
    dl, dh = t - table[lo], table[hi] - t
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    if not signed:
        code = torch.where((t > 0) & (code == 0), 1, code)
    code = torch.where(fin, code, 0x7F)
    if signed:
        code = code | torch.where(torch.signbit(x), 0x80, 0)
    return code.to(torch.uint8), byte.to(torch.uint8)


# ------------------------------------------------------------------ CPU: refusals
@pytest.fixture(scope="module")
def lib():
    from diff_gaussian_rasterization import _C

    return _C.load_library()


def _err(lib):
    return lib.gsr_last_error().decode()


def test_select_rows_abi_refusals(lib):
    f = lib.gsr_select_rows
    assert f(1, None, -1, 1, 1, 1, None) != 0 and "bad P" in _err(lib)
    assert f(1, None, 4, -1, 1, 1, None) != 0 and "budget" in _err(lib)
    assert f(None, None, 4, 2, 1, 1, None) != 0 and "NULL" in _err(lib)
    assert f(1, None, 4, 2, None, 1, None) != 0 and f(1, None, 4, 2, 1, None, None) != 0
    assert f(None, None, 0, 5, None, None, None) == 0 and f(None, None, 5, 0, None, None, None) == 0
    assert lib.gsr_select_rows_scratch_bytes(0) == 0 == lib.gsr_select_rows_scratch_bytes(-3)
    assert lib.gsr_select_rows_scratch_bytes(1) > 0


def test_take_rows_abi_refusals(lib):
    from diff_gaussian_rasterization import _C

    S = _C.GsrRowsSegment
    assert ctypes.sizeof(S) == 48
    f = lambda seg, n=1, P=4, rows=1, K=2: lib.gsr_take_rows((S * 1)(seg), n, P, rows, K, None)  # noqa: E731
    ok = (1, 1, None, None, 12, 0, 0)
    assert f(ok, n=-1) != 0 and "segment list" in _err(lib)
    assert f(ok, P=-1) != 0 and "bad P" in _err(lib)
    assert f(ok, P=1 << 32) != 0 and "bad P" in _err(lib)
    assert f(ok, K=-1) != 0 and f(ok, K=1 << 31) != 0 and "K" in _err(lib)
    assert f(ok, rows=None) != 0 and "NULL" in _err(lib)
    assert f((None,) + ok[1:]) != 0 and "NULL" in _err(lib)
    assert f((1, None) + ok[2:]) != 0 and "NULL" in _err(lib)
    assert f(ok[:5] + (3, 0)) != 0 and "kind" in _err(lib)
    assert f(ok[:4] + (-1, 0, 0)) != 0 and "rows of" in _err(lib)
    assert f(ok[:4] + (1 << 30, 0, 0)) != 0 and "rows of" in _err(lib)
    assert f(ok[:4] + (1 << 20, 0, 0), K=1 << 15) != 0 and "rows of" in _err(lib)
    assert f(ok[:5] + (1, 0)) != 0 and "NULL" in _err(lib)  # codes without scales
    assert f(ok, K=0) == 0 and lib.gsr_take_rows(None, 0, 4, 1, 2, None) == 0
    assert f((None, None, None, None, 0, 0, 0)) == 0  # rows of nothing


def test_python_refusals_on_cpu():
    import train_ops

    with pytest.raises(RuntimeError, match="GPU"):
        train_ops.select_rows(torch.zeros(4), 2)
    with pytest.raises(RuntimeError, match="GPU"):
        train_ops.take_rows([torch.zeros(4)], torch.zeros(2, dtype=torch.int64))


def test_plain_forms_agree_on_cpu():
    """The two oracles of this file on a case worked by hand."""
    s = torch.tensor([1.0, math.nan, 3.0, -0.0, 3.0, 0.0, math.inf, -math.inf])
    assert _select(s, 4) == [0, 2, 4, 6]
    assert _select(s, 2) == [2, 6]
    assert _select(s, 5) == [0, 2, 3, 4, 6]  # -0 and +0 are equal: the first
    assert _select(s, 8) == list(range(8)) and _select(s, 7) == [0, 2, 3, 4, 5, 6, 7]
    pr = torch.tensor([False, True, False, False, False, False, False, True])
    assert _select(s, 1, pr) == [1] and _select(s, 3, pr) == [1, 6, 7]
    code, byte = _encode(torch.tensor([1.0, -1.0625, 2.0 ** -17, 2.0 ** -18]).double(), True)
    assert byte.tolist() == [120]  # 1 -> 128 units of 2^-7
    assert code.tolist() == [0x70, 0xF0, 0, 0]  # 136 is half-way between 128 and 144; 2^-10, 2^-11 are half a step and less
    assert _encode(torch.tensor([1.0, 2.0 ** -30]).double(), False)[0].tolist() == [0x70, 1]


# ------------------------------------------------------------------ GPU: selection
def _scores(kind, P, g):
    if kind == "ties":
        return torch.randint(0, 4, (P,), generator=g).float() * torch.where(torch.rand(P, generator=g) < 0.5, -1.0, 1.0)
    if kind == "equal":
        return torch.full((P,), 2.5)
    if kind == "odd":
        pool = torch.tensor([math.nan, -math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 1.0, -1.0, 3.4e38])
        return pool[torch.randint(0, len(pool), (P,), generator=g)]
    if kind == "close":  # keys that differ in their last bits only
        return (torch.randint(0, 3000, (P,), generator=g, dtype=torch.int32) + 0x3F800000).view(torch.float32)
    return torch.randn(P, generator=g) * torch.exp(8 * torch.randn(P, generator=g))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "odd", "close"])
@pytest.mark.parametrize("P", [1, 2, 5, 64, 1023, 4096, 4097, 20_001])
def test_select_rows_exact(dev, P, kind):
    import train_ops

    g = torch.Generator().manual_seed(P)
    s = _scores(kind, P, g)
    for protect in (None, torch.rand(P, generator=g) < 0.1, torch.ones(P, dtype=torch.bool)):
        for budget in sorted({0, 1, 2, P // 3, P // 2, P - 1, P, P + 7}):
            flat = torch.empty(P + 1, device=dev)  # the scores at an odd element
            flat[1:] = s.to(dev)
            rows = train_ops.select_rows(flat[1:], budget, None if protect is None else protect.to(dev))
            assert rows.dtype == torch.int64
            assert rows.tolist() == _select(s, budget, protect), (budget, protect is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [16_384, 16_385, 300_000, 5_000_011, 17_000_003])
def test_select_rows_large(dev, P):
    import train_ops

    g = torch.Generator(device=dev).manual_seed(1)
    s = torch.exp(2 * torch.randn(P, generator=g, device=dev)) * (torch.rand(P, generator=g, device=dev) < 0.6)
    protect = torch.rand(P, generator=g, device=dev) < 0.01
    x = s.masked_fill(protect, math.inf)
    for budget in (1, P // 10, P // 2, P - P // 5, P - 1):  # also inside the zeros, which are ties
        want = torch.sort(x, descending=True, stable=True).indices[:budget].sort().values
        got = train_ops.select_rows(s.view(P, 1), budget, protect)
        assert torch.equal(got, want), budget


# ------------------------------------------------------------------ GPU: rows
def _raw(t):
    return t.contiguous().view(torch.uint8) if t.dim() else t


@pytest.mark.gpu
@pytest.mark.parametrize("P,K", [(1, 1), (7, 3), (1000, 1), (1000, 999), (1000, 2500), (4096, 4096), (3, 0), (70_001, 60_000)])
def test_take_rows_any_type_and_width(dev, P, K):
    """Rows of 1 to 1028 bytes of many types (more than one launch takes), indices in any order,
    repeated and outside [0, P)."""
    import train_ops

    g = torch.Generator().manual_seed(P + K)
    shapes = [(torch.float32, (3,)), (torch.float32, (1, 3)), (torch.float32, (15, 3)), (torch.float32, (1,)),
              (torch.float32, (4,)), (torch.float32, ()), (torch.float32, (257,)), (torch.bfloat16, (3,)),
              (torch.float16, (8,)), (torch.float64, (2,)), (torch.int64, ()), (torch.uint8, (3,)), (torch.bool, ()),
              (torch.int32, (0, 3)), (torch.uint8, (16,)), (torch.float64, (1,))] * 4
    shapes = shapes if P < 5000 else shapes[:16]
    ts = []
    for dt, s in shapes:
        x = torch.randint(0, 2 if dt is torch.bool else 250, (P, *s), generator=g)
        ts.append(x.to(dt).to(dev))
    odd = torch.randint(0, 250, (P * 12 + 4,), generator=g).to(torch.uint8).to(dev)
    ts.append(odd[4:].view(torch.float32).view(P, 3))  # at 4 bytes
    ts.append(torch.randn(3, P, generator=g).to(dev).t())  # strided
    rows = torch.randint(0, P, (K,), generator=g)
    out = torch.rand(K, generator=g)
    rows = torch.where(out < 0.05, torch.tensor([-1, P, 1 << 40, -(1 << 62)])[torch.randint(0, 4, (K,), generator=g)], rows)
    before = [t.clone() for t in ts]
    got = train_ops.take_rows(ts, rows.to(dev))
    bad = ((rows < 0) | (rows >= P)).to(dev)
    for t, b, q in zip(ts, before, got):
        assert torch.equal(_raw(t), _raw(b))  # bytes: some of them are NaN
        want = t[rows.to(dev).clamp(0, P - 1)].clone()
        want[bad] = 0
        assert q.shape == want.shape and q.dtype == want.dtype and q.is_contiguous()
        assert torch.equal(_raw(q), _raw(want)), (t.dtype, t.shape)


def _state8(shape, seed, dev, spread=6.0):
    """A state whose blocks lie far apart, with zeros."""
    g = torch.Generator().manual_seed(seed)
    n = math.prod(shape)
    nb = -(-n // 64)
    st = {"step": 3}
    for k, signed in (("exp_avg", True), ("exp_rms", False)):
        codes = torch.randint(0, 0x79, (n,), generator=g)
        codes = torch.where(torch.rand(n, generator=g) < 0.1, 0, codes)
        if signed:
            codes = codes | torch.where(torch.rand(n, generator=g) < 0.5, 0x80, 0)
        scale = (100 + spread * torch.randn(nb, generator=g)).clamp(0, 247)
        st[k] = codes.to(torch.uint8).view(shape).view(torch.float8_e4m3fn).to(dev)
        st[k + "_scale"] = scale.to(torch.uint8).view(torch.float8_e8m0fnu).to(dev)
    return st


@pytest.mark.gpu
@pytest.mark.parametrize("P,K", [(1, 1), (9, 5), (64, 64), (1000, 777), (333, 1500), (20_003, 9_999)])
@pytest.mark.parametrize("spread", [0.0, 6.0, 40.0])
def test_take_rows_of_8_bit_states(dev, P, K, spread):
    import train_ops

    g = torch.Generator().manual_seed(K)
    widths = [(3,), (1, 3), (15, 3), (1,), (), (4,), (0, 3), (64,), (130,)]
    states = [_state8((P, *w), k, dev, spread) for k, w in enumerate(widths)]
    nanat = states[0]["exp_avg"].view(torch.uint8)
    nanat[0, 0] = 0x7F
    ordered = torch.randperm(P, generator=g)[:K].sort().values
    for rows in (ordered, torch.where(torch.rand(K, generator=g) < 0.1, -1, torch.randint(0, P, (K,), generator=g))):
        _, got = train_ops.take_rows([], rows.to(dev), states)
        for st, q, w in zip(states, got, widths):
            assert q["step"] == 3
            for key, signed in (("exp_avg", True), ("exp_rms", False)):
                x = _values(st[key].cpu(), st[key + "_scale"].cpu())[rows.clamp(0, P - 1)]
                x[(rows < 0) | (rows >= P)] = 0.0
                code, byte = _encode(x, signed)
                assert q[key].shape == (len(rows), *w) and q[key].dtype == torch.float8_e4m3fn
                assert torch.equal(q[key + "_scale"].cpu().view(torch.uint8), byte), (w, key)
                have = q[key].cpu().view(torch.uint8).reshape(-1)
                nan = code & 0x7F == 0x7F
                assert torch.equal(have[~nan], code[~nan]) and bool((have[nan] & 0x7F == 0x7F).all()), (w, key)


@pytest.mark.gpu
def test_take_rows_all_rows_in_order_keeps_8_bit_values(dev):
    """Every row in place: values as they were (a block's codes may move to another scale), for
    values of 2^-13 of their block's largest and more: 2^-6 units of 128."""
    import train_ops

    st = _state8((501, 45), 1, dev, 0.0)
    for k in ("exp_avg", "exp_rms"):
        c = st[k].view(torch.uint8)
        c[(c & 0x7F) < 0x10] = 0  # below 2^-5: half the units under a scale twice as large
    _, (got,) = train_ops.take_rows([], torch.arange(501, device=dev), [st])
    for k in ("exp_avg", "exp_rms"):
        a = train_ops.unpack_state8(st[k], st[k + "_scale"])
        b = train_ops.unpack_state8(got[k], got[k + "_scale"])
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_take_rows_beyond_32_bit_offsets(dev):
    import train_ops

    P = 70_000_001  # 64-byte rows: 4.5 GB
    t = torch.zeros(P, 16, device=dev)
    rows = torch.tensor([P - 1, 0, P - 2, 67_108_864, P], device=dev)
    t[rows[:4]] = torch.arange(1, 65, device=dev, dtype=torch.float32).view(4, 16)
    (got,) = train_ops.take_rows([t], rows)
    assert torch.equal(got[:4], t[rows[:4]]) and not got[4].any()
    del t, got
    big = torch.arange(P, device=dev)  # many rows out: 2^32 bytes and more of them
    src = torch.arange(64, device=dev, dtype=torch.float32).view(1, 64).repeat(3, 1)
    (got,) = train_ops.take_rows([src], (big % 3)[:17_000_000])
    assert torch.equal(got[-5:], src[:1].expand(5, 64)) and torch.equal(got[:5], src[:1].expand(5, 64))


@pytest.mark.gpu
def test_rows_refusals_on_gpu(dev):
    import train_ops

    s, r = torch.zeros(8, device=dev), torch.zeros(3, dtype=torch.int64, device=dev)
    for kw, exc, msg in [(dict(score=s.half(), budget=1), RuntimeError, "float32"), (dict(score=s.view(2, 4), budget=1), RuntimeError, "P"),
                         (dict(score=s, budget=-1), ValueError, "budget"), (dict(score=s, budget=2.0), ValueError, "budget"),
                         (dict(score=s, budget=1, protect=s), RuntimeError, "protect"),
                         (dict(score=s, budget=1, protect=s[:4] > 0), RuntimeError, "protect"),
                         (dict(score=s, budget=1, protect=s.cpu() > 0), RuntimeError, "protect")]:
        with pytest.raises(exc, match=msg):
            train_ops.select_rows(**kw)
    st = train_ops.adamw_state(torch.zeros(8, 3, device=dev), 8)
    for ts, rows, states, msg in [([s], r.int(), None, "int64"), ([s], r.view(1, 3), None, "vector"), ([s], r.cpu(), None, "GPU"),
                                  ([s, s[:4]], r, None, "same number"), ([s, s.cpu()], r, None, "same number"),
                                  ([s.sum()], r, None, "same number"), ([s[:4]], r, [st], "same number"),
                                  ([s], r, [{**st, "exp_rms_scale": st["exp_rms_scale"][:0]}], "exp_rms_scale")]:
        with pytest.raises(RuntimeError, match=msg):
            train_ops.take_rows(ts, rows, states)
    assert train_ops.take_rows([], r) == [] and train_ops.take_rows([], r, []) == ([], [])
    (e,) = train_ops.take_rows([torch.zeros(0, 5, device=dev)], torch.tensor([-1, 0], device=dev))
    assert e.shape == (2, 5) and not e.any()


@pytest.mark.gpu
def test_take_rows_of_conjugate_and_negated_views(dev):
    """Views whose values differ from their bytes."""
    import train_ops

    z = torch.complex(torch.arange(12.0), torch.arange(1.0, 13.0)).view(6, 2).to(dev)
    rows = torch.tensor([4, 0, 4], device=dev)
    ts = [z.conj(), z.conj().imag, z]
    for t, got in zip(ts, train_ops.take_rows(ts, rows)):
        assert torch.equal(torch.view_as_real(got.resolve_conj()) if got.is_complex() else got,
                           torch.view_as_real(t[rows].resolve_conj()) if t.is_complex() else t[rows].resolve_neg())


@pytest.mark.gpu
def test_optimizer_take_rows_keeps_parameters_what_they_are(dev):
    import train_ops

    p, q = torch.nn.Parameter(torch.randn(6, 2, device=dev)), torch.randn(6, device=dev)
    opt = train_ops.FusedAdamW([{"params": [p], "lr": 0.1}, {"params": [q], "lr": 0.1}], state_bits=8)
    p.grad = torch.ones_like(p)
    opt.step()  # q has no state
    rows = torch.tensor([5, 0, 5], device=dev)
    for bad in (torch.ones(3, device=dev), torch.ones(1, dtype=torch.bool, device=dev)):
        with pytest.raises(RuntimeError, match="fresh"):
            opt.take_rows(rows, bad)
    new = opt.take_rows(rows)
    assert isinstance(new[0], torch.nn.Parameter) and new[0].requires_grad and not new[1].requires_grad
    assert torch.equal(new[0], p[rows]) and torch.equal(new[1], q[rows])
    assert list(opt.state) == [new[0]] and opt.param_groups[1]["params"][0] is new[1]
    new[0].grad = torch.ones_like(new[0])
    opt.step()
    assert opt.state[new[0]]["step"] == 2


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Norm, selection and gather on two streams side by side: each call has scratch of its own."""
    import train_ops

    P, K = 200_003, 70_000
    ins = [(torch.rand(P, device=dev), torch.randn(P, 45, device=dev), _state8((P, 3), k, dev)) for k in range(2)]

    def go(score, x, st):
        norm, scale = train_ops.grad_norm([x], 1.0)
        rows = train_ops.select_rows(score, K)
        (y,), (q,) = train_ops.take_rows([x], rows, [st])
        return [norm, scale, rows, y] + [q[k].view(torch.uint8) for k in q if k != "step"]

    want = [go(*i) for i in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(go(*ins[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(a, b) for g in got[k] for a, b in zip(g, want[k]))


@pytest.mark.gpu
def test_select_and_take_captured_and_replayed(dev):
    """Both in one graph (no host wait, the kept count is known), replayed over new scores with
    eager work between, and on a side stream."""
    import train_ops

    P, K = 50_001, 20_000
    score, x = torch.rand(P, device=dev), torch.randn(P, 45, device=dev)
    st = _state8((P, 3), 5, dev)

    def go():
        rows = train_ops.select_rows(score, K)
        return rows, train_ops.take_rows([x], rows, [st])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, ((y,), (q,)) = go()
    for k in range(4):
        score.copy_(torch.rand(P, device=dev))
        x.mul_(1.25)
        er, ((ey,), (eq,)) = go()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows, er) and torch.equal(y, ey), k
        for key in ("exp_avg", "exp_rms", "exp_avg_scale", "exp_rms_scale"):
            assert torch.equal(q[key].view(torch.uint8), eq[key].view(torch.uint8)), (k, key)


# ------------------------------------------------------------------ GPU: together
@pytest.mark.gpu
def test_blend_weight_sums_to_the_image(dev):
    """sum_i score_i = sum over pixels of 1 - T_final: the image of white Gaussians on black.  fp32
    sums of up to 12288 pixels of weights in [0, 1] in any order: within 12288 u of the total."""
    import synthetic
    import train_step

    cam = synthetic.make_camera(128, 96, 0).to(dev)
    bg = torch.zeros(3, device=dev)
    g = synthetic.make_gaussians(3000, 1, seed=0).to(dev, requires_grad=True)
    score = torch.zeros(3000, device=dev)
    train_step.accumulate_blend_weight(cam, g, bg, score)
    with torch.no_grad():
        white = train_step.render(cam, g, bg, override_color=torch.ones(3000, 3, device=dev))["render"][0]
    total = float(white.double().sum())
    assert total > 1 and bool((score >= 0).all())
    assert abs(float(score.double().sum()) - total) <= 12288 * 2.0 ** -24 * total
    assert all(p.grad is None for p in g.params())
    once = score.clone()
    train_step.accumulate_blend_weight(cam, g, bg, score)  # accumulates
    torch.testing.assert_close(score, 2 * once, rtol=1e-3, atol=1e-4)
    with pytest.raises(RuntimeError, match="score"):
        train_step.accumulate_blend_weight(cam, g, bg, score[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_train_evict_train(dev, bits):
    """The path as a user runs it: training steps, the accumulated blending weight of the views, the
    eviction to a budget with optimiser states and statistics, and training on."""
    import synthetic
    import train_ops
    import train_step

    P, budget = 4000, 2501
    cams = [synthetic.make_camera(128, 96, v).to(dev) for v in range(2)]
    target = synthetic.make_target(128, 96, seed=1).to(dev)
    bg = torch.zeros(3, device=dev)
    g = synthetic.make_gaussians(P, 3, seed=0).to(dev, requires_grad=True)
    st = train_step.TrainState(g, spatial_lr_scale=1.0, fused=True, state_bits=bits, max_norm=1.0)
    for it in (1, 2, 3):
        train_step.full_train_step(it, cams[it % 2], g, st, target, bg)
    score = torch.zeros(P, device=dev)
    for c in cams:
        train_step.accumulate_blend_weight(c, g, bg, score)
    protect = torch.zeros(P, dtype=torch.bool, device=dev)
    protect[:10] = True
    old = [p.detach().clone() for p in g.params()]
    states = [st.optimizer.state[p] for p in g.params()]
    stats = [x.clone() for x in (st.xyz_gradient_accum, st.denom, st.max_radii2D)]
    rows = st.prune_to_budget(g, score, budget, protect)
    assert rows.tolist() == _select(score.cpu(), budget, protect.cpu())
    for p, o in zip(g.params(), old):
        assert p.is_leaf and p.requires_grad and p.grad is None and torch.equal(p, o[rows])
    for x, o in zip((st.xyz_gradient_accum, st.denom, st.max_radii2D), stats):
        assert torch.equal(x, o[rows])
    assert all(a is b for a, b in zip([p for gr in st.optimizer.param_groups for p in gr["params"]], g.params()))
    for p, s in zip(g.params(), states):
        q = st.optimizer.state[p]
        assert q["step"] == 3
        if bits == 32:
            assert torch.equal(q["exp_avg"], s["exp_avg"][rows]) and torch.equal(q["exp_avg_sq"], s["exp_avg_sq"][rows])
        else:
            x = train_ops.unpack_state8(s["exp_rms"], s["exp_rms_scale"])[rows]
            y = train_ops.unpack_state8(q["exp_rms"], q["exp_rms_scale"])
            code, byte = _encode(x.double().cpu(), False)
            assert torch.equal(q["exp_rms"].cpu().view(torch.uint8).reshape(-1), code) and y.shape == x.shape
    assert len(st.optimizer.state) == 6
    for it in (4, 5):
        loss = train_step.full_train_step(it, cams[it % 2], g, st, target, bg)
    assert torch.isfinite(loss) and all(torch.isfinite(p).all() for p in g.params())
    # densify: clones take their parents' rows and no history
    K = budget + 3
    rows = torch.cat([torch.arange(budget, device=dev), torch.tensor([5, 5, 7], device=dev)])
    fresh = torch.arange(K, device=dev) >= budget
    before = [st.optimizer.state[p] for p in g.params()]
    new = st.optimizer.take_rows(rows, fresh)
    assert torch.equal(new[0][budget:], new[0][[5, 5, 7]])
    for p, s in zip(new, before):
        q = st.optimizer.state[p]
        second = q["exp_avg_sq"] if bits == 32 else train_ops.unpack_state8(q["exp_rms"], q["exp_rms_scale"])
        assert second.shape[0] == K and not second[budget:].any()
        assert bits == 8 or torch.equal(second[:budget], s["exp_avg_sq"])


@pytest.mark.gpu
def test_prune_needs_the_optimiser_that_moves_states(dev):
    import synthetic
    import train_step

    g = synthetic.make_gaussians(10, 0).to(dev, requires_grad=True)
    st = train_step.TrainState(g, 1.0, fused=True)
    with pytest.raises(RuntimeError, match="FusedAdamW"):
        st.prune_to_budget(g, torch.zeros(10, device=dev), 5)
    st = train_step.TrainState(g, 1.0, fused=True, state_bits=32)
    with pytest.raises(RuntimeError, match="scores"):
        st.prune_to_budget(g, torch.zeros(9, device=dev), 5)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [1000, 20_000])
def test_select_rows_of_a_negated_view(dev, P):
    import train_ops

    s = torch.randn(P, generator=torch.Generator().manual_seed(P))
    got = train_ops.select_rows(torch._neg_view(-s.to(dev)), P // 3)
    assert torch.equal(got.cpu(), torch.tensor(_select(s, P // 3)))


@pytest.mark.gpu
def test_take_rows_of_negated_states(dev):
    import train_ops

    m, rows = torch.randn(50, 3, device=dev), torch.tensor([7, -1, 49], device=dev)
    st = {"step": 1, "exp_avg": torch._neg_view(-m), "exp_avg_sq": m * m}
    _, (got,) = train_ops.take_rows([], rows, [st])
    assert torch.equal(got["exp_avg"][[0, 2]], m[[7, 49]]) and not got["exp_avg"][1].any()
