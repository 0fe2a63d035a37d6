"""The state-space block's operators on the GPU against the float64 oracle (oracle/ssm_oracle.py), element by element: |got - want| <= half a step of
the output's type + the oracle's first-order bound of float32 arithmetic.  `split`: the scan's 16-bit forms cut the operands of its inner products
to two bfloat16 terms (2^-17 of a term at most, two of them in a product)."""
import math

import numpy as np
import pytest

import ssm_oracle as orc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SPLIT = {"f32": 0.0, "bf16": 3 * 2.0**-17, "f16": 3 * 2.0**-17}


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, slack, dtype=None, what=""):
    """Every element within half a step of its type and the oracle's bound; NaN in `want`: no value is promised."""
    half = torch.finfo(got.dtype if dtype is None else dtype).eps / 2
    got = f64(got)
    told = ~np.isnan(want)
    tiny = 2.0**-25 if got.dtype == np.float64 and dtype is None and half == 2.0**-11 else 0.0   # half a step of float16's subnormals
    over = np.abs(got - want)[told] - (half * (np.abs(want) + slack) + slack)[told] - tiny
    assert over.size == 0 or not (over > 0).any(), (what, float(over.max()), int((over > 0).sum()), float(np.abs(got - want)[told].max()))


def normal(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda") * scale


def ssm():
    from mDeepFRI import ssm
    return ssm


def lens_of(kind):
    return {"one": [1], "ones": [1, 1, 1], "tile": [32, 64, 31, 33], "ragged": [5, 0, 130, 1, 64, 63, 65, 0, 17], "long": [301], "cut": [1300, 5, 0, 513, 256]}[kind]


# ---------------------------------------------------------------------------------------------------------------------
def conv_inputs(seed, lens, channels, width, dtype, align=1, kept=False, extra_cols=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = ssm().SequenceRows.build(lens, align=align)
    total = int(rows.row_off[-1])
    wide = normal(g, max(total, 1), channels + extra_cols).to(TYPES[dtype])[:total]
    x = wide[:, extra_cols:]
    weight, bias = normal(g, width, channels), normal(g, channels)
    n = len(lens)
    kw = {}
    if kept:
        kw = dict(state=normal(g, n + 2, width, channels).to(TYPES[dtype]), slots=torch.randperm(n + 2, generator=g, device="cuda")[:n].int(),
                  positions=torch.tensor([(0, 1, 2, 7, 1000)[i % 5] for i in range(n)], dtype=torch.int32, device="cuda"))
    return rows, x, weight, bias, kw


def check_conv(rows, x, weight, bias, kw, silu=True, out=None):
    ref = {k: f64(v) if k == "state" else v.cpu().numpy() for k, v in kw.items()}
    want, slack = orc.conv(f64(x), f64(weight), None if bias is None else f64(bias), silu, rows.lengths.cpu().numpy(), rows.row_off.cpu().numpy(), **ref)
    got = ssm().causal_conv(x, weight, rows, bias=bias, silu=silu, out=out, **kw)
    near(got, want, slack)
    if "state" in kw:
        assert np.array_equal(f64(kw["state"]), ref["state"])
    return got, want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens, channels, width, align, extra", [("one", 1, 4, 1, 0), ("ragged", 64, 4, 16, 0), ("ragged", 72, 3, 1, 8), ("tile", 33, 2, 1, 3), ("ragged", 264, 8, 1, 0),
                                                                 ("long", 520, 4, 1, 0), ("ones", 130, 1, 1, 0)])
def test_conv(dtype, lens, channels, width, align, extra):
    rows, x, weight, bias, kw = conv_inputs(1, lens_of(lens), channels, width, dtype, align, extra_cols=extra)
    check_conv(rows, x, weight, bias, kw)
    check_conv(rows, x, weight, None, kw, silu=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens, channels, width", [("ragged", 64, 4), ("ones", 40, 3), ("tile", 37, 2), ("long", 128, 8), ("ragged", 16, 1)])
def test_conv_keeps_its_state(dtype, lens, channels, width):
    rows, x, weight, bias, kw = conv_inputs(2, lens_of(lens), channels, width, dtype, kept=True)
    check_conv(rows, x, weight, bias, kw)


@pytest.mark.parametrize("dtype, width, total", [("f32", 3, 12400), ("f32", 8, 12400), ("bf16", 4, 12400), ("f16", 7, 20600), ("bf16", 2, 12400)])
def test_conv_of_many_rows_takes_several_tiles_per_thread(dtype, width, total):
    """Sequences that begin and end anywhere in a thread's tiles, some shorter than the kernel is wide, with their states."""
    some = np.random.default_rng(5).choice([0, 1, 2, 3, 7, 8, 9, 31, 70, 500], size=2000)
    lens = some[: int(np.searchsorted(np.cumsum(some), total)) + 1].tolist()
    rows, x, weight, bias, kw = conv_inputs(5, lens, 1024, width, dtype, kept=True)
    check_conv(rows, x, weight, bias, kw)


def test_conv_skips_sequences_and_leaves_other_rows():
    rows, x, weight, bias, kw = conv_inputs(3, [5, 20, 7, 40], 64, 4, "bf16", align=16, kept=True)
    kw["slots"] = torch.tensor([1, -1, 99, 0], dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 7.0)
    got, want = check_conv(rows, x, weight, bias, kw, out=out)
    untouched = torch.from_numpy(np.isnan(want)).cuda()
    assert got is out and bool((out[untouched] == 7).all())
    kw["positions"].zero_()
    made = ssm().causal_conv(x, weight, rows, bias=bias, **kw)
    assert bool((made[untouched] == 0).all()) and not bool((made[~untouched] == 0).all())


def test_conv_non_finite_inputs_stay_where_they_are():
    rows, x, weight, bias, kw = conv_inputs(4, [40, 9], 64, 4, "f32")
    clean = ssm().causal_conv(x, weight, rows, bias=bias)
    x = x.clone()
    x[10, 3], x[44, 5] = math.nan, math.inf
    got = ssm().causal_conv(x, weight, rows, bias=bias)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[10:14, 3], hit[44:48, 5] = True, True
    assert torch.equal(got[~hit], clean[~hit]) and not torch.isfinite(got[hit]).all()


# ---------------------------------------------------------------------------------------------------------------------
def scan_inputs(seed, lens, heads, groups, head_dim, state_dim, dtype, align=1, kept=False, pad=0, dt_dtype=None, strong=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = ssm().SequenceRows.build(lens, align=align)
    total, n = int(rows.row_off[-1]), len(lens)
    hp, gn = heads * head_dim, groups * state_dim
    xbc = normal(g, max(total, 1), pad + hp + 2 * gn).to(TYPES[dtype])[:total, pad:]
    x, b, c = xbc[:, :hp].unflatten(1, (heads, head_dim)), xbc[:, hp:hp + gn].unflatten(1, (groups, state_dim)), xbc[:, hp + gn:].unflatten(1, (groups, state_dim))
    dt = normal(g, max(total, 1), heads)[:total].to(TYPES[dt_dtype or dtype])
    a = -torch.rand(heads, generator=g, device="cuda") * 15 * strong - 1
    kw = dict(d=normal(g, heads), dt_bias=normal(g, heads) - 3)
    if kept:
        kw.update(state=normal(g, n + 2, heads, head_dim, state_dim), slots=torch.randperm(n + 2, generator=g, device="cuda")[:n].int(),
                  positions=torch.tensor([(0, 3, 1)[i % 3] for i in range(n)], dtype=torch.int32, device="cuda"))
    return rows, x, dt, a, b, c, kw


def check_scan(rows, x, dt, a, b, c, kw, out=None):
    ref = {k: f64(v) if v.is_floating_point() else v.cpu().numpy() for k, v in kw.items()}
    split = SPLIT[{v: k for k, v in TYPES.items()}[x.dtype]]
    want, slack, hslack = orc.scan(f64(x), f64(dt), f64(a), f64(b), f64(c), rows.lengths.cpu().numpy(), rows.row_off.cpu().numpy(), split=split, **ref)
    got = ssm().selective_scan(x, dt, a, b, c, rows, out=out, **kw)
    near(got, want, slack, what="y")
    if "state" in kw:
        written = ~np.isnan(hslack)
        near(kw["state"], np.where(written, ref["state"], np.nan), np.where(written, hslack, 0), what="state")
        assert np.array_equal(f64(kw["state"])[~written], ref["state"][~written])
    return got, want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens, heads, groups, head_dim, state_dim, align, pad", [
    ("one", 1, 1, 1, 1, 1, 0), ("ones", 2, 1, 64, 128, 1, 0), ("ragged", 8, 1, 64, 64, 16, 0), ("ragged", 6, 3, 40, 33, 1, 0), ("tile", 4, 2, 32, 16, 1, 8), ("tile", 3, 1, 96, 128, 1, 1),
    ("ragged", 5, 5, 17, 7, 1, 3), ("long", 2, 1, 128, 128, 1, 0), ("long", 2, 2, 256, 100, 1, 0), ("tile", 16, 1, 32, 32, 1, 0),
    ("cut", 2, 1, 32, 64, 1, 0), ("cut", 3, 3, 40, 33, 16, 1), ("cut", 4, 2, 33, 128, 1, 0)])
def test_scan(dtype, lens, heads, groups, head_dim, state_dim, align, pad):
    check_scan(*scan_inputs(11, lens_of(lens), heads, groups, head_dim, state_dim, dtype, align, pad=pad))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens, heads, groups, head_dim, state_dim", [("ragged", 4, 1, 64, 128), ("ones", 6, 3, 40, 33), ("long", 3, 1, 48, 64), ("tile", 1, 1, 20, 128), ("cut", 2, 1, 64, 128), ("cut", 3, 1, 17, 30)])
def test_scan_keeps_its_state(dtype, lens, heads, groups, head_dim, state_dim):
    check_scan(*scan_inputs(12, lens_of(lens), heads, groups, head_dim, state_dim, dtype, kept=True))


def test_scan_without_skip_bias_and_with_other_types_of_dt():
    for dtype, dt_dtype in (("bf16", "f32"), ("f32", "bf16"), ("f16", "f16")):
        rows, x, dt, a, b, c, kw = scan_inputs(13, [70, 3], 4, 1, 32, 24, dtype, dt_dtype=dt_dtype)
        check_scan(rows, x, dt, a, b, c, {})


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("groups, head_dim, state_dim, pad", [(1, 32, 64, 0), (1, 33, 31, 0), (3, 17, 33, 1)])
def test_rows_of_no_sequence_do_not_reach_results(dtype, groups, head_dim, state_dim, pad):
    """Rows between and behind sequences full of NaN, on whole words and off them: outputs and states as with zeros there."""
    lens = [37, 1, 0, 64, 5]
    rows, x, dt, a, b, c, kw = scan_inputs(19, lens, 3, groups, head_dim, state_dim, dtype, align=16, kept=True, pad=pad)
    crows, cx, weight, bias, ckw = conv_inputs(20, lens, 40 + pad, 4, dtype, align=16, kept=True, extra_cols=pad)
    inside = torch.zeros(x.shape[0], dtype=torch.bool, device="cuda")
    for o, n in zip(rows.row_off.tolist(), lens):
        inside[o:o + n] = True
    again = {k: v.clone() for k, v in kw.items()}, {k: v.clone() for k, v in ckw.items()}
    want, cwant = ssm().selective_scan(x, dt, a, b, c, rows, **kw), ssm().causal_conv(cx, weight, crows, bias=bias, **ckw)
    for t in (x, dt, b, c, cx):
        t[~inside] = math.nan
    got, cgot = ssm().selective_scan(x, dt, a, b, c, rows, **again[0]), ssm().causal_conv(cx, weight, crows, bias=bias, **again[1])
    assert torch.equal(got, want) and torch.equal(cgot, cwant) and torch.equal(again[0]["state"], kw["state"]) and torch.equal(again[1]["state"], ckw["state"])
    assert bool((got[~inside] == 0).all()) and bool((cgot[~inside] == 0).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_step_size_of_minus_infinity_masks_its_token(dtype):
    """softplus(-inf) = 0: the token changes no state and reads the one in front of it; the type's lowest value does the same; a row of nothing but such
    tokens gives d x alone."""
    rows, x, dt, a, b, c, kw = scan_inputs(24, [70, 40], 3, 1, 32, 48, dtype)
    dt = dt.clone()
    dt[5:9, 1], dt[64, 0], dt[70:110, 2] = -math.inf, torch.finfo(dt.dtype).min, -math.inf
    got, want = check_scan(rows, x, dt, a, b, c, kw)
    assert torch.isfinite(got).all()
    near(got[70:, 2], f64(x[70:, 2]) * float(kw["d"][2]), np.abs(f64(x[70:, 2])) * 1e-6 + 1e-30)
    xbc, sdt, sa, skw = step_inputs(25, 4, 3, 1, 32, 48, 4, dtype)
    sdt[1] = -math.inf
    check_step(xbc, sdt, sa, skw)


def test_scan_cut_into_segments_skips_sequences_and_spoils_only_what_follows():
    """Sequences longer than a workgroup's share: their segments run side by side and hand their states on.  A skipped one stays as it is, a NaN spoils its
    channel from its token to the sequence's end through every later segment, and the workspace is refused when it is too small."""
    import ctypes
    from mDeepFRI import _hip
    rows, x, dt, a, b, c, kw = scan_inputs(17, [900, 1500, 640], 2, 1, 32, 64, "bf16", kept=True)
    kw["slots"] = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    out = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda")
    got, want = check_scan(rows, x, dt, a, b, c, kw, out=out)
    assert bool((out[900:2400] == 7).all())
    clean = {k: v.clone() for k, v in kw.items()}
    bad = {k: v.clone() for k, v in kw.items()}
    clean_out = ssm().selective_scan(x, dt, a, b, c, rows, **clean)
    spoilt = x.clone()
    spoilt[300, 1, 9] = math.nan
    out = ssm().selective_scan(spoilt, dt, a, b, c, rows, **bad)
    hit = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    hit[300:900, 1, 9] = True
    assert torch.equal(out[~hit], clean_out[~hit]) and not torch.isfinite(out[hit]).any()
    state_hit = torch.zeros_like(bad["state"], dtype=torch.bool)
    state_hit[1, 1, 9] = True
    assert torch.equal(bad["state"][~state_hit], clean["state"][~state_hit]) and not torch.isfinite(bad["state"][state_hit]).any()
    g = ssm()._Scan()
    g.dtype = g.dt_dtype = _hip.DT_BF16
    g.heads, g.groups, g.head_dim, g.state_dim, g.ldx, g.ldb, g.ldc, g.lddt, g.ldy = 2, 1, 32, 64, x.stride(0), b.stride(0), c.stride(0), dt.stride(0), 64
    g.x, g.b, g.c, g.dt, g.a, g.y = x.data_ptr(), b.data_ptr(), c.data_ptr(), dt.data_ptr(), a.data_ptr(), out.data_ptr()
    g.rows.lengths, g.rows.row_off, g.rows.R, g.rows.B, g.rows.max_len = rows.lengths.data_ptr(), rows.row_off.data_ptr(), x.shape[0], 3, rows.max_len
    need = _hip.lib().mdf_scan_workspace_bytes(ctypes.byref(g))
    assert need > 0 and _hip.lib().mdf_selective_scan_dev(ctypes.byref(g), None, 0, None) == _hip.MDF_ECAPACITY
    with pytest.raises(_hip.CapacityError, match="workspace"):
        _hip.check(_hip.lib().mdf_selective_scan_dev(ctypes.byref(g), out.data_ptr(), need - 1, None))


def test_scan_with_a_longest_length_that_is_too_short():
    """max_len sizes the cut only: a longer sequence is still run to its end, states and all."""
    rows, x, dt, a, b, c, kw = scan_inputs(18, [1700, 600], 2, 1, 32, 64, "f32", kept=True)
    rows.max_len = 700
    check_scan(rows, x, dt, a, b, c, kw)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_with_decays_that_forget_at_once(dtype):
    """Log-decays of hundreds per token: everything but the last tokens underflows, nothing overflows on the way."""
    rows, x, dt, a, b, c, kw = scan_inputs(14, [200, 33], 4, 1, 32, 64, dtype, strong=40.0)
    kw["dt_bias"] = kw["dt_bias"] + 6
    check_scan(rows, x, dt, a, b, c, kw)


def test_scan_skips_sequences_and_leaves_other_rows():
    rows, x, dt, a, b, c, kw = scan_inputs(15, [5, 50, 7, 40], 4, 1, 32, 64, "bf16", align=16, kept=True)
    kw["slots"] = torch.tensor([4, -1, 6, 0], dtype=torch.int32, device="cuda")
    out = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda")
    got, want = check_scan(rows, x, dt, a, b, c, kw, out=out)
    untouched = torch.from_numpy(np.isnan(want)).cuda()
    assert bool((out[untouched] == 7).all())
    junk = torch.full_like(x, math.nan)
    del junk                                             # what the allocator hands out next is full of NaN
    made = ssm().selective_scan(x, dt, a, b, c, rows, **kw)
    assert bool((made[untouched] == 0).all()) and torch.isfinite(made).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_scan_non_finite_values_stay_where_the_recurrence_puts_them(dtype, value):
    """A bad x spoils its channel from its token on, a bad c its token, a bad b its group's heads from its token on, a bad dt its head from its token
    on; every other value keeps its bits."""
    lens = [100, 40]
    rows, x, dt, a, b, c, kw = scan_inputs(16, lens, 4, 2, 32, 48, dtype)
    clean = ssm().selective_scan(x, dt, a, b, c, rows, **kw)
    for name in ("x", "c", "b", "dt"):
        t = {"x": x.clone(), "b": b.clone(), "c": c.clone(), "dt": dt.clone()}
        hit = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
        if name == "x":
            t["x"][45, 1, 7], hit[45:100, 1, 7] = value, True
        elif name == "c":
            t["c"][45, 1, 5], hit[45, 2:] = value, True
        elif name == "b":
            t["b"][45, 1, 5], hit[45:100, 2:] = value, True
        else:
            t["dt"][45, 3], hit[45:100, 3] = value, True
        got = ssm().selective_scan(t["x"], t["dt"], a, t["b"], t["c"], rows, **kw)
        assert torch.equal(got[~hit], clean[~hit]), name
        assert not torch.isfinite(got[hit]).any(), name


# ---------------------------------------------------------------------------------------------------------------------
def step_inputs(seed, n, heads, groups, head_dim, state_dim, width, dtype, pool=3, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ch = heads * head_dim + 2 * groups * state_dim
    kw = dict(conv_weight=normal(g, width, ch) * width**-0.5, conv_bias=normal(g, ch, scale=0.1), conv_state=normal(g, n + pool, width, ch).to(TYPES[dtype]),
              state=normal(g, n + pool, heads, head_dim, state_dim), slots=torch.randperm(n + pool, generator=g, device="cuda")[:n].int(),
              positions=torch.tensor([(5, 0, 1, 2, 1000, 3)[i % 6] for i in range(n)], dtype=torch.int32, device="cuda"), d=normal(g, heads), dt_bias=normal(g, heads) - 3)
    xbc = normal(g, n, ch + pad).to(TYPES[dtype])[:, pad:]
    return xbc, normal(g, n, heads).to(TYPES[dtype]), -torch.rand(heads, generator=g, device="cuda") * 15 - 1, kw


def check_step(xbc, dt, a, kw, out=None):
    heads, head_dim, state_dim = kw["state"].shape[1:]
    groups = (xbc.shape[1] - heads * head_dim) // (2 * state_dim)
    n, hp, gn = xbc.shape[0], heads * head_dim, groups * state_dim
    ref = {k: None if v is None else f64(v) if v.is_floating_point() else v.cpu().numpy() for k, v in kw.items()}
    slots = ref["slots"] if ref["slots"] is not None else np.arange(n)
    live = np.array([0 <= s < len(ref["state"]) for s in slots])
    ones, off = [1] * n, np.arange(n + 1)
    u, us = orc.conv(f64(xbc), ref["conv_weight"], ref["conv_bias"], True, ones, off, ref["conv_state"], slots, ref["positions"])
    u, us = np.nan_to_num(u), np.nan_to_num(us)
    part = lambda v: (v[:, :hp].reshape(n, heads, head_dim), v[:, hp:hp + gn].reshape(n, groups, state_dim), v[:, hp + gn:].reshape(n, groups, state_dim))  # noqa: E731
    x, b, c = part(u)
    dx, db, dc = part(us)
    old = ref["state"].copy()
    want, slack, hslack = orc.scan(x, f64(dt), f64(a), b, c, ones, off, ref["d"], ref["dt_bias"], ref["state"], slots, ref["positions"])
    rep = np.arange(heads) // (heads // groups)
    v = f64(dt) + ref["dt_bias"]
    delta = (np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v))))[:, :, None]
    new = np.stack([ref["state"][s] if ok else old[0] for s, ok in zip(slots, live)])
    dh = delta[..., None] * (dx[..., None] * np.abs(b[:, rep])[:, :, None] + np.abs(x)[..., None] * db[:, rep][:, :, None])       # what the convolution's own error does to the state
    slack = slack + (dh * np.abs(c[:, rep])[:, :, None] + np.abs(new) * dc[:, rep][:, :, None]).sum(-1) + np.abs(ref["d"])[:, None] * dx
    for i, (s, ok) in enumerate(zip(slots, live)):
        if ok:
            hslack[s] += dh[i]
    got = ssm().selective_step(xbc, dt, a, out=out, **kw)
    near(got, want, slack, what="y")
    written = ~np.isnan(hslack)
    near(kw["state"], np.where(written, ref["state"], np.nan), np.where(written, hslack, 0), what="state")
    assert np.array_equal(f64(kw["state"])[~written], ref["state"][~written])
    assert np.array_equal(f64(kw["conv_state"]), ref["conv_state"])
    return got, want


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n, heads, groups, head_dim, state_dim, width, pad", [(1, 1, 1, 1, 1, 1, 0), (1, 8, 1, 64, 128, 4, 0), (7, 6, 3, 40, 33, 3, 0), (33, 4, 2, 64, 64, 4, 5), (3, 2, 1, 256, 128, 8, 0),
                                                                             (130, 3, 1, 96, 16, 2, 0), (5, 2, 2, 17, 100, 4, 3)])
def test_step(dtype, n, heads, groups, head_dim, state_dim, width, pad):
    check_step(*step_inputs(21, n, heads, groups, head_dim, state_dim, width, dtype, pad=pad))


def test_step_skips_a_padded_batch():
    xbc, dt, a, kw = step_inputs(22, 6, 4, 1, 32, 64, 4, "bf16")
    kw["slots"] = torch.tensor([3, -1, 0, 9, 8, -5], dtype=torch.int32, device="cuda")
    out = torch.full((6, 4, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    before = {k: v.clone() for k, v in kw.items()}
    check_step(xbc, dt, a, kw, out=out)
    assert bool((out[[1, 3, 5]] == 7).all())
    made = ssm().selective_step(xbc, dt, a, **before)
    assert torch.equal(made[[0, 2, 4]], out[[0, 2, 4]]) and bool((made[[1, 3, 5]] == 0).all())


def test_step_in_a_pool_whose_offsets_pass_32_bits():
    """A state behind element 2^31 of the pool (8.7 GB)."""
    heads, head_dim, state_dim, width, slots = 32, 64, 128, 4, 8300
    xbc, dt, a, kw = step_inputs(23, 2, heads, 1, head_dim, state_dim, width, "bf16")
    small = {k: v.clone() for k, v in kw.items()}
    small["slots"] = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    want = ssm().selective_step(xbc, dt, a, **small)
    pool, ring = torch.empty(slots, heads, head_dim, state_dim, device="cuda"), torch.zeros(slots, width, xbc.shape[1], dtype=xbc.dtype, device="cuda")
    for i, s in enumerate((8299, 8193)):
        pool[s], ring[s] = kw["state"][i], kw["conv_state"][i]
    kw.update(state=pool, conv_state=ring, slots=torch.tensor([8299, 8193], dtype=torch.int32, device="cuda"))
    assert torch.equal(ssm().selective_step(xbc, dt, a, **kw), want)
    assert torch.equal(pool[[8299, 8193]], small["state"][:2]) and torch.equal(ring[[8299, 8193]], small["conv_state"][:2])


# ---------------------------------------------------------------------------------------------------------------------
def norm_inputs(seed, rows, dim, dtype, residual, gate, post, pre, center, scale_vec):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[dtype]
    kw = dict(center=center, eps=1e-5)
    if gate:
        kw["gate"] = normal(g, rows, dim).to(t)
    if residual:
        kw.update(residual=normal(g, rows, dim, scale=3).to(torch.float32 if residual == "f32" else t), scale=0.7)
        if scale_vec:
            kw["scale_vec"] = torch.rand(dim, generator=g, device="cuda")
    for k, on in (("post", post), ("pre", pre)):
        if on:
            kw[k + "_weight"] = 1 + normal(g, dim, scale=0.2)
            if center:
                kw[k + "_bias"] = normal(g, dim, scale=0.2)
    return (normal(g, rows, dim) + (2 if center else 0)).to(t), kw


def check_norm(s, kw, **outs):
    want_r, want = orc.block_norm(f64(s), **{k: f64(v) if torch.is_tensor(v) else v for k, v in kw.items()})
    r, o = ssm().block_norm(s, **kw, **outs)
    assert (r is None) == (want_r is None) and (o is None) == (want is None)
    if r is not None:
        near(r, *want_r, what="residual")
    if o is not None:
        near(o, *want, what="out")
    return r, o


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows, dim", [(1, 1), (3, 64), (5, 100), (33, 513), (17, 1024), (9, 2048), (4, 5001), (2, 32768)])
def test_norm_forms(dtype, rows, dim):
    for i, (residual, gate, first, act, post, pre, center, vec) in enumerate([
            (None, True, True, "silu", True, False, False, False), (None, False, False, "silu", True, False, True, False), (None, False, False, "silu", False, True, False, False),
            ("f32", True, False, "sigmoid", True, True, False, True), ("same", False, False, "silu", False, True, True, True), ("same", True, True, "none", True, False, False, False),
            ("f32", True, False, "silu", False, False, False, False), (None, True, False, "silu", True, True, False, False)]):
        s, kw = norm_inputs(31 + i, rows, dim, dtype, residual, gate, post, pre, center, vec)
        check_norm(s, dict(kw, gate_first=first, gate_act=act))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [512, 520, 1025, 2049, 4096, 4097, 8192, 8193, 16384, 16385])
def test_norm_widths(dtype, dim):
    """The widths on both sides of each change of threads per row."""
    for i, (residual, gate, post, pre, center, vec) in enumerate([(None, True, True, False, False, False), ("f32", True, True, True, True, True), ("same", False, True, True, False, False)]):
        s, kw = norm_inputs(61 + i, 3, dim, dtype, residual, gate, post, pre, center, vec)
        check_norm(s, dict(kw, gate_first=i == 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim, groups", [(64, 8), (1024, 4), (999, 3), (2048, 2), (24, 24)])
def test_norm_groups(dtype, dim, groups):
    s, kw = norm_inputs(41, 13, dim, dtype, None, True, True, False, False, False)
    check_norm(s, dict(kw, groups=groups, gate_first=True))
    s, kw = norm_inputs(42, 13, dim, dtype, "f32", True, True, False, True, True)
    check_norm(s, dict(kw, groups=groups))


def test_norm_in_place_strides_and_broadcast_rows():
    s, kw = norm_inputs(43, 20, 520, "bf16", "f32", True, True, True, False, True)
    r, o = ssm().block_norm(s, **kw)
    wide = torch.zeros(20, 1100, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:523] = s
    res = kw["residual"].clone()
    r2, o2 = ssm().block_norm(wide[:, 3:523], **dict(kw, residual=res), residual_out=res, out=wide[:, 3:523])     # both outputs in place, rows unaligned
    assert r2 is res and torch.equal(res, r) and torch.equal(wide[:, 3:523], o) and bool((wide[:, :3] == 0).all()) and bool((wide[:, 523:] == 0).all())
    one = kw["gate"][:1].expand(20, 520)                                                                   # one gate for every row
    want, _ = ssm().block_norm(s, **dict(kw, gate=one.contiguous()))
    got, _ = ssm().block_norm(s, **dict(kw, gate=one))
    assert torch.equal(got, want)


def test_norm_of_rows_without_anything_and_of_non_finite_ones():
    """A row of zeros gives zeros (eps), a row with a NaN or an infinity spoils itself alone."""
    s, kw = norm_inputs(44, 6, 300, "f32", "f32", False, True, True, False, False)
    clean = ssm().block_norm(s, **kw)
    s = s.clone()
    s[1], s[3, 7], s[4, 299] = 0, math.nan, math.inf
    r, o = ssm().block_norm(s, **kw)
    keep = [0, 2, 5]
    assert torch.equal(r[keep], clean[0][keep]) and torch.equal(o[keep], clean[1][keep])
    assert torch.equal(r[1], kw["residual"][1]) and torch.isfinite(o[1]).all()
    assert not torch.isfinite(o[3]).any() and not torch.isfinite(o[4]).all()
    z, _ = ssm().block_norm(torch.zeros(3, 300, device="cuda"), post_weight=kw["post_weight"])[1], None
    assert bool((z == 0).all())


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
def block_weights(seed, dim, heads, groups, head_dim, state_dim, width):
    g = torch.Generator(device="cuda").manual_seed(seed)
    inner, gn = heads * head_dim, groups * state_dim
    return dict(heads=heads, groups=groups, head_dim=head_dim, state_dim=state_dim, inner=inner, gn=gn, pre=1 + normal(g, dim, scale=0.1), post=1 + normal(g, dim, scale=0.1),
                mid=1 + normal(g, inner, scale=0.1), w_in=normal(g, dim, 2 * inner + 2 * gn + heads, scale=dim**-0.5), w_out=normal(g, inner, dim, scale=inner**-0.5),
                conv=normal(g, width, inner + 2 * gn, scale=width**-0.5), conv_bias=normal(g, inner + 2 * gn, scale=0.1), a=-torch.rand(heads, generator=g, device="cuda") * 8 - 1,
                d=normal(g, heads), dt_bias=normal(g, heads, scale=0.5) - 3)


def run_block(w, hidden, mixer):
    """One block over rows `hidden` (f32 residual stream); `mixer(xbc, dt)` is the convolution and the scan."""
    S = ssm()
    _, n = S.block_norm(hidden, post_weight=w["pre"])
    zxbcdt = n @ w["w_in"]
    z, xbc, dt = zxbcdt[:, :w["inner"]], zxbcdt[:, w["inner"]:-w["heads"]], zxbcdt[:, -w["heads"]:]
    y = mixer(xbc, dt).flatten(1)
    _, y = S.block_norm(y, gate=z, gate_first=True, post_weight=w["mid"])
    return S.block_norm(y @ w["w_out"], residual=hidden, post_weight=w["post"], scale=0.5)[0]


def test_block_of_prompts_then_tokens_equals_whole_prompts():
    """A batch of prompts through the whole block in one call == prompts cut short, the rest token by token through the kept states (f32: the same
    sums in another order)."""
    S = ssm()
    w = block_weights(51, 96, 4, 2, 32, 48, 4)
    lens, cut = [40, 7, 65, 33], [37, 1, 60, 33]
    g = torch.Generator(device="cuda").manual_seed(52)
    hidden = [normal(g, n, 96) for n in lens]
    split = lambda u: (u[:, :w["inner"]].unflatten(1, (4, 32)), u[:, w["inner"]:w["inner"] + w["gn"]].unflatten(1, (2, 48)), u[:, w["inner"] + w["gn"]:].unflatten(1, (2, 48)))  # noqa: E731

    def prompts(rows, **kept):
        conv_kept = dict(state=kept["ring"]) if kept else {}

        def mixer(xbc, dt):
            x, b, c = split(S.causal_conv(xbc, w["conv"], rows, bias=w["conv_bias"], **conv_kept))
            return S.selective_scan(x, dt, w["a"], b, c, rows, d=w["d"], dt_bias=w["dt_bias"], **(dict(state=kept["state"]) if kept else {}))
        return mixer

    whole = run_block(w, torch.cat(hidden), prompts(S.SequenceRows.build(lens)))
    ring, state = torch.zeros(4, 4, w["inner"] + 2 * w["gn"], device="cuda"), torch.zeros(4, 4, 32, 48, device="cuda")
    first = run_block(w, torch.cat([h[:k] for h, k in zip(hidden, cut)]), prompts(S.SequenceRows.build(cut), ring=ring, state=state))
    got = [list(p) for p in first.split(cut)]
    positions = torch.tensor(cut, dtype=torch.int32, device="cuda")
    for t in range(max(n - k for n, k in zip(lens, cut))):
        on = [i for i in range(4) if cut[i] + t < lens[i]]
        slots = S.check_slots([i if i in on else -1 for i in range(4)], 4)
        rows = torch.stack([hidden[i][min(cut[i] + t, lens[i] - 1)] for i in range(4)])
        out = run_block(w, rows, lambda xbc, dt: S.selective_step(xbc, dt, w["a"], conv_weight=w["conv"], conv_bias=w["conv_bias"], conv_state=ring, state=state, positions=positions,
                                                                  slots=slots, d=w["d"], dt_bias=w["dt_bias"]))
        for i in on:
            got[i].append(out[i])
        positions += 1
    got = torch.cat([torch.stack(p) for p in got])
    assert float((got - whole).abs().max()) < 2e-4 * float(whole.abs().max())     # some 2000 float32 operations deep, each within 2^-24 of values of the largest's size


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_and_replayed_with_other_inputs(dtype):
    """Every operator in one graph; replays see new inputs in the same buffers and give the eager results' bits, with eager work between them."""
    S = ssm()
    rows, x, dt, a, b, c, kw = scan_inputs(61, [70, 1, 33], 4, 1, 32, 64, dtype, kept=True)
    total, ch = x.shape[0], 4 * 32 + 2 * 64
    src = torch.empty(total, ch, dtype=TYPES[dtype], device="cuda")
    _, _, weight, bias, ckw = conv_inputs(62, [70, 1, 33], ch, 4, dtype, kept=True)
    sx, sdt, sa, skw = step_inputs(63, 3, 4, 1, 32, 64, 4, dtype)

    def everything(kw, ckw, skw):
        u = S.causal_conv(src, weight, rows, bias=bias, **ckw)
        y = S.selective_scan(u[:, :128].unflatten(1, (4, 32)), dt, a, u[:, 128:192].unflatten(1, (1, 64)), u[:, 192:].unflatten(1, (1, 64)), rows, **kw)
        _, n = S.block_norm(y.flatten(1), gate=u[:, :128], gate_first=True, post_weight=torch.ones(128, device="cuda") if False else ones)
        return u, y, n, S.selective_step(src[:3], sdt, sa, **skw)

    ones = torch.ones(128, device="cuda")
    fresh = lambda d: {k: v.clone() for k, v in d.items()}  # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(64)
    k1, k2, k3 = fresh(kw), fresh(ckw), fresh(skw)
    src.copy_(normal(g, total, ch).to(src.dtype))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        everything(fresh(kw), fresh(ckw), fresh(skw))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = everything(k1, k2, k3)
    e1, e2, e3 = fresh(kw), fresh(ckw), fresh(skw)      # capture ran nothing: the states are still the first ones
    for _ in range(4):
        src.copy_(normal(g, total, ch).to(src.dtype))
        graph.replay()
        want = everything(e1, e2, e3)
        torch.cuda.synchronize()
        for got, w in zip(outs + (k1["state"], k2["state"], k3["state"], k3["conv_state"]), want + (e1["state"], e2["state"], e3["state"], e3["conv_state"])):
            assert torch.equal(got, w)


def test_on_another_stream_than_the_tensors_own():
    S = ssm()
    rows, x, dt, a, b, c, kw = scan_inputs(71, [300, 40], 4, 1, 64, 128, "bf16")
    want = S.selective_scan(x, dt, a, b, c, rows, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = S.selective_scan(x, dt, a, b, c, rows, **kw)
        done = got.clone()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(done, want)


def test_same_inputs_same_bits():
    S = ssm()
    rows, x, dt, a, b, c, kw = scan_inputs(72, [700, 40, 350], 8, 2, 64, 128, "bf16")
    want = S.selective_scan(x, dt, a, b, c, rows, **kw)
    for _ in range(3):
        assert torch.equal(S.selective_scan(x, dt, a, b, c, rows, **kw), want)


def test_refusals_on_the_device():
    S = ssm()
    rows, x, dt, a, b, c, kw = scan_inputs(81, [10, 5], 4, 2, 32, 16, "bf16")
    with pytest.raises(ValueError, match="one type"):
        S.selective_scan(x, dt, a, b.float(), c, rows)
    with pytest.raises(ValueError, match="only the row stride"):
        S.selective_scan(x.transpose(1, 2).contiguous().transpose(1, 2), dt, a, b, c, rows)
    with pytest.raises(ValueError, match="inference only"):
        S.selective_scan(x.clone().requires_grad_(), dt, a, b, c, rows)
    with pytest.raises(ValueError, match="kept state"):
        S.selective_scan(x, dt, a, b, c, rows, positions=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="float32"):
        S.selective_scan(x, dt, a.double(), b, c, rows)
    with pytest.raises(ValueError, match="overlaps"):
        S.selective_scan(x, dt, a, b, c, rows, out=x)
    with pytest.raises(ValueError, match="shape"):
        S.selective_scan(x, dt[:, :3], a, b, c, rows)
    with pytest.raises(ValueError, match="state_dim"):
        S.selective_scan(x, dt, a, torch.zeros(15, 2, 129, dtype=x.dtype, device="cuda"), torch.zeros(15, 2, 129, dtype=x.dtype, device="cuda"), rows)
    with pytest.raises(ValueError, match="int32"):
        S.causal_conv(x.flatten(1), torch.zeros(4, 128, device="cuda"), rows, state=torch.zeros(2, 4, 128, dtype=x.dtype, device="cuda"), slots=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with torch.no_grad():
        S.selective_scan(x.clone().requires_grad_(), dt, a, b, c, rows)
