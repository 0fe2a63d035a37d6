"""The state-space block's operators on the GPU in calls at the edges of what their documentation allows."""
import numpy as np
import pytest

import ssm_oracle as orc
from test_gpu_ssm import TYPES, check_scan, f64, near, scan_inputs, ssm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---------------------------------------------------------------------------------------------------------------------
# 16-bit outputs are float32 results, rounded once
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scan_reads_a_state_to_its_last_bit(dtype):
    """Masked tokens (D = 0) whose c picks one entry of the state: y is that float32 number, rounded once to the output's type -- no arithmetic in between is
    inexact, so every bit counts."""
    heads, head_dim, state_dim, n = 4, 64, 32, 3
    rows, x, dt, a, b, c, _ = scan_inputs(201, [state_dim] * n, heads, 1, head_dim, state_dim, dtype)
    g = torch.Generator(device="cuda").manual_seed(202)
    state = torch.randn(n, heads, head_dim, state_dim, generator=g, device="cuda")
    c = torch.eye(state_dim, device="cuda").repeat(n, 1).to(x.dtype).unsqueeze(1).contiguous()
    positions = torch.ones(n, dtype=torch.int32, device="cuda")
    got = ssm().selective_scan(x, torch.full_like(dt, -np.inf), a, b, c, rows, state=state, positions=positions)
    want = state.permute(0, 3, 1, 2).reshape(got.shape).to(x.dtype)
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens, state_dim", [([1] * 300, 2), ([1, 3, 2, 4] * 60, 4)])
def test_scan_rounds_as_float32_arithmetic_does(dtype, lens, state_dim):
    """Where the oracle's value less and plus its bound of float32 arithmetic round to the same number, every float32 result in between does: the output is that
    number."""
    rows, x, dt, a, b, c, kw = scan_inputs(203, lens, 4, 1, 64, state_dim, dtype)
    want, slack, _ = orc.scan(f64(x), f64(dt), f64(a), f64(b), f64(c), rows.lengths.cpu().numpy(), rows.row_off.cpu().numpy(), d=f64(kw["d"]), dt_bias=f64(kw["dt_bias"]))
    got = ssm().selective_scan(x, dt, a, b, c, rows, **kw).cpu()
    low, high = (torch.from_numpy(v).to(TYPES[dtype]) for v in (want - slack, want + slack))
    told = low == high
    assert float(told.double().mean()) > 0.9
    assert torch.equal(got[told], low[told]), int((got[told] != low[told]).sum())


# ---------------------------------------------------------------------------------------------------------------------
# rows of no sequence
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens, longer", [([5, 40, 1], 100), ([7], 1), ([], 33), ([0, 0], 5)])
def test_rows_behind_the_last_sequence_are_zero_in_an_output_made_here(dtype, lens, longer):
    """An array longer than the sequences in it (a buffer of one size for every batch), while the allocator hands out memory full of NaN."""
    total = sum(lens) + longer
    _, x, dt, a, b, c, kw = scan_inputs(211, [total], 3, 1, 32, 48, dtype)
    rows = ssm().SequenceRows.build(lens)
    assert rows.dense
    weight = torch.ones(4, 96, device="cuda")
    for call in (lambda: ssm().selective_scan(x, dt, a, b, c, rows, **kw), lambda: ssm().causal_conv(x.flatten(1), weight, rows).view(x.shape)):
        junk = torch.full(x.shape, np.nan, dtype=x.dtype, device="cuda")
        del junk
        got = call()
        assert bool((got[sum(lens):] == 0).all()) and bool(torch.isfinite(got).all())
        assert sum(lens) == 0 or bool((got[:sum(lens)] != 0).any())


def test_a_residual_scale_changed_in_place_is_the_one_used():
    s, r = torch.ones(3, 64, device="cuda"), torch.zeros(3, 64, device="cuda")
    scale = torch.tensor(0.5)
    for k in (0.5, 0.25, -3.0):
        scale.fill_(k)
        got, _ = ssm().block_norm(s, residual=r, scale=scale)
        assert bool((got == k).all())
    with pytest.raises(ValueError, match="host"):
        ssm().block_norm(s, residual=r, scale=scale.cuda())


# ---------------------------------------------------------------------------------------------------------------------
# long sequences among short ones
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [[2600] + [1] * 40, [1] * 300 + [2100] + [0] * 5 + [1] * 200, [255, 256, 257, 0, 511, 512, 513, 768, 0, 0, 1025, 1, 256, 769], [1, 1400, 3, 1200, 0, 257, 2]])
def test_scan_cuts_long_sequences_among_short_ones(dtype, lens):
    """Lengths on both sides of whole segments, behind any number of short and empty sequences, with states that begin and continue."""
    check_scan(*scan_inputs(221, lens, 2, 1, 32, 24, dtype, kept=True))


def test_scan_cuts_a_long_sequence_among_more_sequences_than_a_grid_is_high():
    rows, x, dt, a, b, c, kw = scan_inputs(222, [1] * 70000 + [1500], 1, 1, 32, 8, "f32")
    got = ssm().selective_scan(x, dt, a, b, c, rows, **kw)
    alone = ssm().SequenceRows.build([1500])
    last = lambda t: t[70000:]  # noqa: E731
    want, slack, _ = orc.scan(f64(last(x)), f64(last(dt)), f64(a), f64(last(b)), f64(last(c)), [1500], [0], d=f64(kw["d"]), dt_bias=f64(kw["dt_bias"]))
    near(last(got), want, slack)
    near(ssm().selective_scan(last(x), last(dt), a, last(b), last(c), alone, **kw), want, slack)
    once = ssm().SequenceRows.build([1] * 70000)
    assert torch.equal(got[:70000], ssm().selective_scan(x[:70000], dt[:70000], a, b[:70000], c[:70000], once, **kw))


# ---------------------------------------------------------------------------------------------------------------------
# more rows than one dimension of a grid holds
# ---------------------------------------------------------------------------------------------------------------------
def same_rows(got, make, rows, step=1 << 24):
    """`got` against make(slice) piece by piece (a whole float64 copy would be large)."""
    for r in range(0, rows, step):
        at = slice(r, min(r + step, rows))
        want, slack = make(at)
        assert bool(((got[at].double() - want).abs() <= slack).all()), r


def test_norm_of_2_to_26_rows():
    """Per-head norms of a long batch: 64 threads a row pass 2^32 threads."""
    rows, dim = 2**26 + 5, 4
    g = torch.Generator(device="cuda").manual_seed(231)
    s = torch.randn(rows, dim, generator=g, device="cuda")
    w = torch.tensor([1.0, 2.0, 0.5, -1.0], device="cuda")
    _, got = ssm().block_norm(s, post_weight=w, eps=1e-6)

    def make(at):
        v = s[at].double()
        want = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * w.double()
        return want, want.abs() * 16 * 2.0**-24 + 1e-36      # a sum of 4 squares, a mean, a root, a division and two products
    same_rows(got, make, rows)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_of_rows_in_several_launches_in_place(dtype):
    """Gate, residual and both outputs in place over 2^21 + 3 rows: each row as by itself."""
    rows, dim = 2**21 + 3, 24
    g = torch.Generator(device="cuda").manual_seed(232)
    s, gate = (torch.randn(rows, dim + 8, generator=g, device="cuda").to(TYPES[dtype])[:, 8:] for _ in range(2))
    res = torch.randn(rows, dim, generator=g, device="cuda")
    kw = dict(post_weight=torch.rand(dim, generator=g, device="cuda"), pre_weight=torch.rand(dim, generator=g, device="cuda"), scale=0.5)
    some = [0, 1, 2**21 - 1, 2**21, 2**21 + 1, 2**21 + 2]
    want_r, want = ssm().block_norm(s[some], gate=gate[some], residual=res[some], **kw)
    half = ssm().block_norm(s[2**20:], gate=gate[2**20:], residual=res[2**20:], **kw)
    r, out = ssm().block_norm(s, gate=gate, residual=res, residual_out=res, out=s, **kw)
    assert torch.equal(r[some], want_r) and torch.equal(out[some], want)
    assert torch.equal(r[2**20:], half[0]) and torch.equal(out[2**20:], half[1])


def test_scan_of_2_to_24_sequences():
    """One-row sequences, a workgroup each: y = (c b D + d) x."""
    n = 2**24 + 9
    g = torch.Generator(device="cuda").manual_seed(233)
    x, b, c = (torch.randn(n, 1, 1, generator=g, device="cuda") for _ in range(3))
    dt, a = torch.randn(n, 1, generator=g, device="cuda"), torch.tensor([-1.0], device="cuda")
    lengths, off = torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    got = ssm().selective_scan(x, dt, a, b, c, ssm().SequenceRows(lengths, off, 1, dense=True))

    def make(at):
        want = c[at].double() * b[at].double() * torch.nn.functional.softplus(dt[at].double(), threshold=100).unsqueeze(2) * x[at].double()
        return want, want.abs() * 40 * 2.0**-24 + 1e-36      # softplus 12 + |dt| steps and the products' dropped terms
    same_rows(got, make, n)


def test_step_of_2_to_24_sequences():
    """Width 1 without a bias: u = silu(w xbc), y = u_c u_b D u_x, in their own states and in chosen ones."""
    n = 2**24 + 3
    g = torch.Generator(device="cuda").manual_seed(234)
    xbc, dt = torch.randn(n, 3, generator=g, device="cuda"), torch.randn(n, 1, generator=g, device="cuda")
    w, a = torch.tensor([[1.0, -2.0, 0.5]], device="cuda"), torch.tensor([-1.0], device="cuda")
    ring, state = torch.full((n, 1, 3), 7.0, device="cuda"), torch.full((n, 1, 1, 1), 7.0, device="cuda")
    got = ssm().selective_step(xbc, dt, a, conv_weight=w, conv_state=ring, state=state).clone()

    def parts(at):
        u = w.double() * xbc[at].double()
        u = u * torch.sigmoid(u)
        h = torch.nn.functional.softplus(dt[at].double(), threshold=100) * u[:, :1] * u[:, 1:2]
        return u, h

    def make(at):
        u, h = parts(at)
        want = (h * u[:, 2:]).unsqueeze(2)
        return want, want.abs() * 100 * 2.0**-24 + 1e-36     # three silu of 8 + 2 |u| steps, |u| < 12, a softplus of 12 + |dt|, three products
    same_rows(got, make, n)
    same_rows(state, lambda at: (parts(at)[1].view(-1, 1, 1, 1), parts(at)[1].abs().view(-1, 1, 1, 1) * 80 * 2.0**-24 + 1e-36), n)
    assert torch.equal(ring[:, 0], xbc)
    slots = torch.arange(n - 1, -1, -1, dtype=torch.int32, device="cuda")
    again, ring2, state2 = ssm().selective_step, torch.zeros_like(ring), torch.zeros_like(state)
    assert torch.equal(again(xbc, dt, a, conv_weight=w, conv_state=ring2, state=state2, slots=slots), got)
    assert torch.equal(state2.flip(0), state) and torch.equal(ring2.flip(0), ring)


def test_a_tangent_is_refused_in_a_call_of_a_known_form():
    """What is kept of an earlier call's checks must not let it through."""
    from torch.autograd import forward_ad
    rows, x, dt, a, b, c, kw = scan_inputs(241, [9, 4], 2, 1, 32, 16, "f32")
    want = ssm().selective_scan(x, dt, a, b, c, rows, **kw)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="dt carries a tangent"):
            ssm().selective_scan(x, forward_ad.make_dual(dt, torch.ones_like(dt)), a, b, c, rows, **kw)
        assert torch.equal(ssm().selective_scan(x, dt, a, b, c, rows, **kw), want)
    assert torch.equal(ssm().selective_scan(x, dt, a, b, c, rows, **kw), want)


# ---------------------------------------------------------------------------------------------------------------------
# values at the ends of the range
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_scan_with_step_sizes_around_the_smallest_float32(dtype):
    """softplus of -80 to -110: normal, subnormal and 0; every other token an ordinary one."""
    rows, x, dt, a, b, c, kw = scan_inputs(251, [130, 64], 3, 1, 32, 48, dtype)
    dt = dt.clone()
    dt[::2] = -80 - 30 * torch.arange(dt[::2].numel(), device="cuda").view_as(dt[::2]).float().remainder(31).div(31).to(dt.dtype)
    kw.pop("dt_bias")
    got, _ = check_scan(rows, x, dt, a, b, c, kw)
    assert bool(torch.isfinite(got).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_masked_token_that_is_not_finite_spoils_what_the_recurrence_says(dtype):
    """0 times a NaN is one: a mask is for tokens of finite x and b.  What is not finite in x spoils its channel from there on, beside and before it nothing."""
    rows, x, dt, a, b, c, kw = scan_inputs(252, [70], 3, 1, 32, 48, dtype)
    dt, spoilt = dt.clone(), x.clone()
    dt[40] = -np.inf
    clean = ssm().selective_scan(x, dt, a, b, c, rows, **kw)
    spoilt[40, 1, 3] = np.nan
    got = ssm().selective_scan(spoilt, dt, a, b, c, rows, **kw)
    hit = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    hit[40:, 1, 3] = True
    assert torch.equal(got[~hit], clean[~hit]) and bool(torch.isnan(got[hit]).all())


def test_scan_of_float32_products_leans_to_no_side():
    """y = c h, one product per output (masked tokens, c of one entry).  What the split operands leave out is less than 2^-22 of the product and of either sign, and the
    terms' sum rounds to nearest, so the mean of 2^17 signed relative errors has a standard deviation below 2^-22 / 2^8.5 = 2^-30.5; 2^-27 is eleven of them.  (Terms
    that are all cut off towards zero leave some 2^-24.6.)"""
    g = torch.Generator(device="cuda").manual_seed(261)
    heads, head_dim, state_dim, n = 8, 256, 2, 64
    rows, x, dt, a, b, _, _ = scan_inputs(262, [1] * n, heads, 1, head_dim, state_dim, "f32")
    state = torch.randn(n, heads, head_dim, state_dim, generator=g, device="cuda")
    c = torch.randn(n, 1, state_dim, generator=g, device="cuda")
    c[:, :, 1] = 0
    got = ssm().selective_scan(x, torch.full_like(dt, -np.inf), a, b, c, rows, state=state.clone(), positions=torch.ones(n, dtype=torch.int32, device="cuda"))
    want = c[:, :, 0].double().unsqueeze(2) * state[..., 0].double()
    error = (got.double() - want) / want
    assert error.numel() == 2**17 and float(error.abs().max()) < 2.0**-21
    mean = float(error.mean())
    assert abs(mean) < 2.0**-27, mean


# ---------------------------------------------------------------------------------------------------------------------
# large arrays, replayed graphs
# ---------------------------------------------------------------------------------------------------------------------
def test_rows_behind_32_bit_offsets():
    """Sequences at the end of arrays of more than 2^32 bytes and 2^31 values: the same bits as in an array of their own."""
    S, lens, R = ssm(), [600, 3], 1_050_000
    g = torch.Generator(device="cuda").manual_seed(271)
    heads, head_dim, state_dim = 32, 64, 64
    ch, n = heads * head_dim, sum(lens)
    small = torch.randn(n, ch, generator=g, device="cuda").bfloat16()
    bc, dt = torch.randn(n, 2, state_dim, generator=g, device="cuda").bfloat16(), torch.randn(n, heads, generator=g, device="cuda")
    a, weight, gain = -torch.rand(heads, generator=g, device="cuda") * 4 - 1, torch.randn(4, ch, generator=g, device="cuda"), torch.rand(ch, generator=g, device="cuda")
    big, out = torch.zeros(R, ch, dtype=torch.bfloat16, device="cuda"), torch.empty(R, ch, dtype=torch.bfloat16, device="cuda")
    big[R - n:] = small
    big_bc, big_dt = torch.zeros(R, 2, state_dim, dtype=torch.bfloat16, device="cuda"), torch.zeros(R, heads, device="cuda")
    big_bc[R - n:], big_dt[R - n:] = bc, dt
    own = S.SequenceRows.build(lens)
    far = S.SequenceRows(own.lengths, own.row_off + (R - n), own.max_len)
    heads_of = lambda t: t.view(-1, heads, head_dim)  # noqa: E731
    want = S.selective_scan(heads_of(small), dt, a, bc[:, :1], bc[:, 1:], own).flatten(1)
    S.selective_scan(heads_of(big), big_dt, a, big_bc[:, :1], big_bc[:, 1:], far, out=heads_of(out))
    slack = 2.0**-7 * want.float().abs() + 2e-5 * float(want.float().abs().max())      # cut into other segments: float32 sums in another order may round to the next bfloat16
    assert bool(((out[R - n:].float() - want.float()).abs() <= slack).all())
    want = S.causal_conv(small, weight, own)
    S.causal_conv(big, weight, far, out=out)
    assert torch.equal(out[R - n:], want)
    _, want = S.block_norm(small, post_weight=gain)
    S.block_norm(big, post_weight=gain, out=out)
    assert torch.equal(out[R - n:], want)


def test_a_captured_scan_replayed_with_other_lengths():
    """The cut is sized on the host by max_len; which rows are whose is read on the GPU: one graph for every mix of lengths in the same rows, with eager work and other
    graphs' workspaces between the replays."""
    S = ssm()
    R = 2100
    _, x, dt, a, b, c, kw = scan_inputs(281, [R], 2, 1, 32, 48, "f32")
    mixes = [[2000, 60, 40], [700, 1400, 0], [3, 900, 1197], [0, 0, 2100], [100, 100, 100]]
    lengths, off = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    rows = S.SequenceRows(lengths, off, 2100)
    call = lambda: S.selective_scan(x, dt, a, b, c, rows, **kw)  # noqa: E731

    def fill(lens):
        own = S.SequenceRows.build(lens)
        lengths.copy_(own.lengths), off.copy_(own.row_off)

    fill(mixes[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call())
    for lens in mixes + mixes[::-1]:
        fill(lens)
        for graph in graphs:
            graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager)
        assert bool((eager[sum(lens):] == 0).all())
        want, slack, _ = orc.scan(f64(x), f64(dt), f64(a), f64(b), f64(c), lens, off.tolist(), d=f64(kw["d"]), dt_bias=f64(kw["dt_bias"]))
        near(eager, want, slack)


@pytest.mark.parametrize("dim", [64, 2048, 32768])
def test_norm_of_equal_values_is_one(dim):
    """Rows of k, k, k, ...: squares, sums, mean and root are exact (k <= 256 and a power of two of them: partial sums stay below 2^24 times a power of two), so the
    quotient is 1 to the last bit, which k times a rounded 1 / k is not for one k in seven."""
    k = torch.arange(1, 257, device="cuda").float()
    s = (k * torch.tensor([1.0, -1.0], device="cuda").repeat(128)).unsqueeze(1).expand(256, dim).contiguous()
    w = torch.rand(dim, device="cuda") + 0.5
    _, got = ssm().block_norm(s, post_weight=w, eps=0.0)
    assert torch.equal(got, torch.sign(s) * w)
    r, got = ssm().block_norm(s, residual=torch.zeros_like(s), pre_weight=w, eps=0.0)
    assert torch.equal(r, s) and torch.equal(got, torch.sign(s) * w)


def test_norm_of_rows_whose_squares_leave_the_range_is_no_nan():
    """Mean square infinite: 0, as 1 / infinity says; an infinity among the values is a NaN in its own place."""
    s = torch.full((2, 128), 1e30, device="cuda")
    s[1, 5] = np.inf
    _, got = ssm().block_norm(s, post_weight=torch.ones(128, device="cuda"))
    assert bool((got[0] == 0).all()) and bool(torch.isnan(got[1, 5])) and bool((got[1, :5] == 0).all()) and bool((got[1, 6:] == 0).all())
