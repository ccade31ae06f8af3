"""The serving operators where their inputs reach the ends of what the entries accept: zero points beyond four bits, scales that
lie far apart, rows whose squares vanish in 32 bits, empty extents, non-finite rows, the status word under capture."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from . import serving_reference as ref  # noqa: E402
from .test_serving_gpu import CACHE, E4M3, I8, BF16, F16, F32, _check_attention, _check_norm, _check_w4, _cuda, _gen, _paged, _w4_case, ops  # noqa: E402,F401


# ---- zero points ------------------------------------------------------------------------------------

@pytest.mark.parametrize("m", [1, 5, 12, 40, 130])
@pytest.mark.parametrize("n,k,group", [(77, 1024, 128), (130, 1056, 32), (300, 2048, 32), (256, 1088, 64)])
@pytest.mark.parametrize("dtype", [BF16, F16, E4M3, I8])
def test_w4_zero_points_beyond_four_bits(ops, m, n, k, group, dtype):
    """0 .. 127 are exact: 16 is what formats that store a zero point less one in four bits decode to."""
    d, out = _w4_case(m, n, k, dtype, group, True, True, 1, F32, out_dtype=F32)
    d["zeros"] = torch.randint(0, 128, d["zeros"].shape, generator=_gen(m + n), dtype=torch.uint8)
    d["zeros"].view(-1)[::7] = 16
    d["zeros"].view(-1)[::11] = 127
    _check_w4(ops, d, out)


@pytest.mark.parametrize("m", [1, 12, 40])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_every_zero_point_and_nibble(ops, m, dtype, group):
    """x one-hot and scales of 1: q - z comes back exactly (in f32) up to 127; a zero point above is NaN in its row and in no other."""
    n, k = 256, 512
    q = torch.randint(0, 256, (n, k // 2), generator=_gen(m), dtype=torch.uint8)
    zeros = torch.arange(n, dtype=torch.uint8)[:, None].repeat(1, k // group)
    zeros[:128, 0] = 127 - zeros[:128, 0]  # another zero point in one of the groups
    scales = torch.ones(n, k // group)
    w = ref.w4_weights(q, scales, zeros, group)
    for at in (0, 33, 300, k - m):
        x = torch.zeros(m, k, dtype=dtype)
        x[torch.arange(m), at + torch.arange(m)] = 1.0
        got = ops.w4_matmul(x.cuda(), q.cuda(), scales.cuda(), zeros=zeros.cuda(), group=group, out_dtype=F32).cpu()
        assert torch.equal(got[:, :128].double(), w[:128, at:at + m].t())
        assert torch.isnan(got[:, 128:]).all()


@pytest.mark.parametrize("m", [3, 12, 20, 64])
@pytest.mark.parametrize("n,k,group", [(100, 256, 64), (100, 256, 128), (70, 512, 32)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_w4_a_non_finite_value_reaches_its_whole_row_and_no_other(ops, m, n, k, group, dtype, bad):
    """inf * (q - z) is infinite, or NaN where q = z, and so is every sum that it enters."""
    d, out = _w4_case(m, n, k, dtype, group, True, True, 0, dtype)
    d["x"][m // 2, k // 3] = bad
    got = ops.w4_matmul(**{a: v.cuda() if isinstance(v, torch.Tensor) else v for a, v in d.items()}).cpu()
    rest = torch.arange(m) != m // 2
    assert not torch.isfinite(got[~rest]).any() and torch.isfinite(got[rest]).all()


@pytest.mark.parametrize("x_groups", [0, 1])
def test_w4_no_columns_of_eight_bits(ops, x_groups):
    """K = 0: the bias alone, whether x_scale has a column for each row or one for each of no groups."""
    bias = torch.randn(7, device="cuda", dtype=BF16)
    got = ops.w4_matmul(torch.empty(3, 0, dtype=I8, device="cuda"), torch.empty(7, 0, dtype=torch.uint8, device="cuda"),
                        torch.empty(7, 0, dtype=BF16, device="cuda"), bias=bias, x_scale=torch.ones(3, x_groups, device="cuda"))
    assert got.dtype == BF16 and torch.equal(got, bias.expand(3, 7))


# ---- rms-norm ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,cols", [(3, 64), (5, 1000), (2, 2501), (700, 256), (601, 1537), (3, 8192), (2, 16384), (2, 40000), (3, 3002)])
@pytest.mark.parametrize("eps", [0.0, 2.0**-130, 2.0**-100])
@pytest.mark.parametrize("out,group", [(None, 0), (E4M3, 0), (I8, 64)])
def test_rmsnorm_rows_whose_squares_vanish(ops, rows, cols, eps, out, group):
    """Squares of rows below 2^-75 are nothing in f32, yet with an eps as small the result is near 1."""
    g = _gen(cols)
    x, r = (torch.randn(rows, cols, generator=g) for _ in range(2))
    size = torch.tensor([1e-25, 1e-18, 1e-36, 1e-30, 1.0, 1e-22, 1e18])[torch.arange(rows) % 7][:, None]
    w = torch.rand(cols, generator=g) + 0.5
    _check_norm(ops, x * size, w, None, eps, out, group)
    _check_norm(ops, x * size, None, r * size, eps, out, group)
    _check_norm(ops, (x * size).to(BF16), w.to(BF16), (r * size).to(BF16), eps, out, group)
    one = torch.zeros(rows, cols)
    one[:, cols // 2] = 2.0**-140  # a subnormal alone in its row: sqrt(cols) without eps
    _check_norm(ops, one, None, None, eps, out, group)


def test_rmsnorm_the_largest_values(ops):
    x = torch.full((4, 640), 3e38)
    x[1] = torch.randn(640, generator=_gen(1)) * 1e37
    x[2, 1:] = 1.0
    for shape in ((4, 640), (2, 1280), (1, 2560)):
        at = x.view(shape)
        _check_norm(ops, at, None, None, 1e-6, None, 0)
        _, want = ref.rmsnorm(at, None, None, 1e-6)
        for out, group in ((E4M3, 0), (I8, 64)):
            y, scale, _ = ops.rmsnorm(at.cuda(), out_dtype=out, group=group)
            # the ones beside 3e38 come to less than 2^-119, and groups below that hold zeros: they are off by themselves
            tiny = ref.spread_scale(ref.group_max(want, group), shape[1], group) < 2.0**-119
            y, scale, slack = y.cpu(), scale.cpu().double(), (shape[1] / 16 + 16) * 2.0**-24
            assert (y.float()[tiny] == 0).all()
            s = ref.spread_scale(scale, shape[1], group)
            step = 0.5 * s if out == I8 else torch.maximum(want.abs() * 2.0**-4, s * 2.0**-10)
            assert (((y.double() * s - want).abs() <= step + want.abs() * slack * 2) | tiny).all()
            top = ref.group_max(want, group) / ref.TOP[out]
            assert ((scale - top).abs() <= top * slack + 1e-45).all()


def test_rmsnorm_a_zero_row_without_eps_is_not_a_number(ops):
    x = torch.randn(5, 320, generator=_gen(2))
    x[3] = 0
    for wide in (x, x.repeat(1, 60)):
        y, _, _ = ops.rmsnorm(wide.cuda(), eps=0.0)
        assert torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 2, 4]]).all()


@pytest.mark.parametrize("out", [E4M3, I8])
def test_rmsnorm_rows_without_columns_have_the_scale_zero(ops, out):
    for rows in (1, 5, 3000):
        garbage = torch.full((rows, 1), float("nan"), device="cuda")
        del garbage  # the scale takes its memory
        y, scale, _ = ops.rmsnorm(torch.empty(rows, 0, device="cuda", dtype=BF16), out_dtype=out)
        assert y.shape == (rows, 0) and scale.shape == (rows, 1) and (scale == 0).all()
        _, scale, _ = ops.rmsnorm(torch.empty(rows, 0, device="cuda", dtype=BF16), out_dtype=out, group=64)
        assert scale.shape == (rows, 0)


# ---- append: a block that fills token by token ------------------------------------------------------

@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("block", [16, 64])
def test_append_values_held_and_rounded_again_stay_near_what_was_appended(ops, held, dtype, block):
    """Against the values themselves: a value is off by half a step when it is held and by half a step more for every growth of its block's scale
    since, a step being the scale (int8), or 2^-3 of the value and at least 2^-9 of the scale (e4m3); 2^-20 of the value more for the 32-bit arithmetic."""
    heads, dim, n = 2, 64, block + block // 2
    d = _paged(80, [1], [n], heads, dim, block, dtype, held)
    dev = _cuda(d)
    x = {c: torch.randn(n, heads, dim, generator=_gen(i)).to(dtype) * torch.linspace(0.2, 3.0, n)[:, None, None].to(dtype) for i, c in enumerate("kv")}
    off = {c: torch.zeros(n, heads, dim, dtype=torch.float64) for c in "kv"}
    scales = {c: torch.zeros(heads, dtype=torch.float64) for c in "kv"}
    for i in range(n):
        ops.kv8_append(x["k"][i:i + 1].cuda(), x["v"][i:i + 1].cuda(), *(dev[c] for c in CACHE), dev["block_table"], torch.tensor([i + 1], dtype=torch.int32).cuda())
        page, first = int(d["block_table"][0, i // block]), i // block * block
        for c in "kv":
            now = dev[c + "_scale"][page].cpu().double()
            grew = (now != scales[c]) if i > first else torch.ones(heads, dtype=torch.bool)
            for t in range(first, i + 1):
                size = x[c][t].double().abs() + off[c][t]  # what is rounded
                half = 0.5 * now[:, None] if held == I8 else torch.maximum(size * 2.0**-4, now[:, None] * 2.0**-10)
                off[c][t] += torch.where((grew | (t == i))[:, None], half + size * 2.0**-20, torch.zeros(()))
            scales[c] = now
            got = dev[c + "_cache"][page].cpu().double() * now[:, None, None]
            wrong = (got[:, :i + 1 - first].transpose(0, 1) - x[c][first:i + 1].double()).abs()
            assert (wrong <= off[c][first:i + 1]).all(), (i, (wrong / off[c][first:i + 1]).max())


# ---- attention: value scales that lie far apart -----------------------------------------------------

def _tight_bound(q, d, scale, window):
    """o in 64 bits and a bound for numerators that are held in 16 bits relative to the largest of the ROW's own: as the reference's
    (2^-11, 2^-18 and twice a score's error of the summed magnitudes, half a step of the result), but with a floor that no value outside the
    row's weights raises.  A numerator p * scale is scaled so that the row's largest lies between 2^10 and 2^14; one that is subnormal in f16
    is off by 2^-25, 2^-35 of the largest, times the 8-bit value (448, 127 at most): for each of the n keys."""
    want, _, bound, _ = ref.attention(q, *(d[c] for c in CACHE), d["block_table"], d["seq_lens"], d["cu_new"], scale, window)
    pages, heads, block, dim = d["k_cache"].shape
    group = q.shape[1] // heads
    for b in range(len(d["seq_lens"])):
        n = int(d["cu_new"][b + 1] - d["cu_new"][b])
        for i in range(n):
            pos, t = int(d["seq_lens"][b]) - n + i, int(d["cu_new"][b]) + i
            at = torch.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            page = d["block_table"][b, at // block].long()
            kk = d["k_cache"][page, :, at % block].double() * d["k_scale"][page].double()[:, :, None]
            v8, vs = d["v_cache"][page, :, at % block].double(), d["v_scale"][page].double()
            p = torch.softmax(torch.einsum("hgd,jhd->hgj", q[t].double().reshape(heads, group, dim), kk) * scale, -1)
            size = (torch.einsum("hgd,jhd->hgj", q[t].double().reshape(heads, group, dim).abs(), kk.abs()) * abs(scale)).amax(-1)
            wrong = size * (dim / 16 + 4) * 2.0**-22 + 2.0**-21
            weight = p * vs.t()[:, None, :]
            spread = torch.einsum("hgj,jhd->hgd", weight, v8.abs())
            floor = weight.amax(-1) * len(at) * ref.TOP[d["v_cache"].dtype] * 2.0**-35
            bound[t] = (spread * (2.0**-11 + 2.0**-18 + 2 * wrong[..., None]) + floor[..., None]).reshape(-1, dim) + want[t].abs() * ref.half_step(q.dtype)
            bound[t] += 2.0**-25 if q.dtype == F16 else 0.0
    return want, bound


def _check_tight(ops, d, q_heads, uniform, scale=None, window=0, q=None, rows=slice(None)):
    dim = d["k_cache"].shape[3]
    scale = dim ** -0.5 if scale is None else scale
    if q is None:
        q = torch.randn(d["k"].shape[0], q_heads, dim, generator=_gen(5)).to(d["k"].dtype)
    dev = _cuda(d)
    got = ops.attention_kv8(q.cuda(), *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"], cu_new=None if uniform else dev["cu_new"], scale=scale,
                            window=window).cpu().double()[rows]
    want, bound = (x[rows] for x in _tight_bound(q, d, scale, window))
    off = (got - want).abs()
    assert (off <= bound).all(), (off / bound).nan_to_num(nan=float("inf")).max()


SHAPES = [(1, 1, 64, F16), (2, 4, 128, BF16), (2, 6, 128, F16), (1, 10, 64, BF16)]


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim,dtype", SHAPES)
@pytest.mark.parametrize("huge", [2.0**28, 1e30, float("inf")])
@pytest.mark.parametrize("room", [20, 1200])
def test_attention_a_page_in_front_of_the_window_costs_nothing(ops, held, heads, group, dim, dtype, huge, room):
    """Blocks of 16 are half a step of keys: the page in front of the window is fetched with the window's first one."""
    for lens, window in (([200, 90], 40), ([211, 215], 36), ([300, 300], 117)):  # the first key is 160, 50; 175, 179; 183
        d = _paged(70, [1, 1], lens, heads, dim, 16, dtype, held, table_blocks=room)
        for b, n in enumerate(lens):
            for blk in range((n - window) // 16):
                d["v_scale"][int(d["block_table"][b, blk])] = huge
        _check_tight(ops, d, heads * group, True, window=window)
        _check_tight(ops, d, heads * group, False, window=window)


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim,dtype", SHAPES)
@pytest.mark.parametrize("huge", [2.0**28, 1e30, float("inf")])
@pytest.mark.parametrize("room", [20, 1200])
def test_attention_a_later_tokens_page_costs_earlier_rows_nothing(ops, held, heads, group, dim, dtype, huge, room):
    for lens in ([97, 97], [209, 17], [113, 241]):  # the last new token begins a block, in the first or second half of a step
        d = _paged(71, [5, 5], lens, heads, dim, 16, dtype, held, table_blocks=room)
        for b, n in enumerate(lens):
            d["v_scale"][int(d["block_table"][b, (n - 1) // 16])] = huge
        d["v_scale"] = d["v_scale"].float()
        earlier = torch.tensor([0, 1, 2, 3, 5, 6, 7, 8])
        _check_tight(ops, d, heads * group, True, rows=earlier)
        _check_tight(ops, d, heads * group, False, rows=earlier)


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim,dtype", SHAPES)
@pytest.mark.parametrize("block", [16, 48])
@pytest.mark.parametrize("uniform", [True, False])
def test_attention_a_page_without_weight_costs_nothing(ops, held, heads, group, dim, dtype, block, uniform):
    """A page of huge values whose keys point away from every query: its weight in the softmax is below 2^-126."""
    for huge in (2.0**28, 2.0**60):
        d = _paged(72, [3, 3], [500, 260], heads, dim, block, dtype, held, table_blocks=1200)
        q = (torch.rand(6, heads * group, dim, generator=_gen(8)) + 0.5).to(dtype)
        for b, n in enumerate((500, 260)):
            for blk in (0, 2, 3, (n - 4) // block - 1):
                page = int(d["block_table"][b, blk])
                d["k_cache"][page] = torch.full(d["k_cache"][page].shape, -100.0).to(held)
                d["k_scale"][page] = 0.5
                d["v_scale"][page] = huge
        _check_tight(ops, d, heads * group, uniform, q=q)


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim,dtype", [(2, 4, 128, BF16), (1, 10, 64, BF16), (2, 5, 128, BF16)])
@pytest.mark.parametrize("new", [1, 2, 4])
def test_attention_value_scales_over_the_whole_range(ops, held, heads, group, dim, dtype, new):
    """Scales from 2^-100 to 2^100, zeros among them, in every order."""
    for seed, room in ((73, 40), (74, 1500), (75, 1500)):
        d = _paged(seed, [new] * 3, [600, 77, 1300], heads, dim, 16, dtype, held, table_blocks=max(room, 90))
        order = torch.rand(d["v_scale"].shape, generator=_gen(seed)) * 200 - 100
        if seed == 74:
            order = order.sort(0).values
        if seed == 75:
            order = order / 4 - 70
        d["v_scale"] = torch.where(torch.rand(order.shape, generator=_gen(seed + 1)) < 0.1, torch.zeros(()), torch.exp2(order))
        _check_tight(ops, d, heads * group, True)
        _check_tight(ops, d, heads * group, False)


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim", [(2, 1, 64), (1, 4, 128), (2, 9, 128)])
def test_attention_of_f16_results_takes_its_numerators_in_two_parts(ops, held, heads, group, dim):
    """Few keys, values that cancel: numerators rounded once to f16 (2^-12 of each) would exceed this bound.  Two parts leave 2^-22 of the summed magnitudes,
    the exponential and a score's rounding 2^-18, each of the n / 16 + 8 sums 2^-22, and the result's own rounding 2^-11 of what is left."""
    lens = [2, 3, 4, 6, 8, 16]
    d = _paged(76, [1] * len(lens), lens, heads, dim, 16, F16, held)
    d["k_scale"] = torch.full_like(d["k_scale"], 1e-3)  # scores of some tenths
    d["v_scale"] = torch.full_like(d["v_scale"], 0.0173)
    q = torch.randn(len(lens), heads * group, dim, generator=_gen(9)).to(F16)
    dev = _cuda(d)
    got = ops.attention_kv8(q.cuda(), *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"]).cpu().double()
    for t, n in enumerate(lens):
        page = int(d["block_table"][t, 0])
        k, v = (d[c + "_cache"][page, :, :n].double() * float(d[c + "_scale"][0, 0]) for c in ("k", "v"))
        p = torch.softmax(torch.einsum("hgd,hjd->hgj", q[t].double().view(heads, group, dim), k) * dim ** -0.5, -1)
        want, spread = (torch.einsum("hgj,hjd->hgd", p, x).reshape(-1, dim) for x in (v, v.abs()))
        off = (got[t] - want).abs()
        bound = spread * (2.0**-22 + 2.0**-18 + (n / 16 + 8) * 2.0**-22) + want.abs() * ref.half_step(F16) + 2.0**-25
        assert (off <= bound).all(), (n, (off / bound).max())


# ---- the status word --------------------------------------------------------------------------------

FIRST_CALL = """
import torch
from intent_ir_b200 import ops
torch.manual_seed(0)
x, q, s = torch.randn(2, 256).to(torch.bfloat16).cuda(), torch.randint(0, 256, (64, 128), dtype=torch.uint8).cuda(), torch.ones(64, 2).cuda()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    gone = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    del gone  # its memory is the pool's again, and every replay writes it
    y = ops.w4_matmul(x, q, s)
    assert ops._status_address(0), "the captured product has no word to report to"
word = ops._status[0]
assert word.data_ptr() == ops._status_address(0)
for _ in range(3):
    graph.replay()
ops.check_device_status()
assert int(word) == 0
want = ops.w4_matmul(x, q, s)
assert torch.equal(y, want) and ops._status[0] is word
word.fill_(8)  # as a wait that ran out would leave it
graph.replay()  # which a replay does not wipe out
try:
    ops.check_device_status()
except ops.B200RuntimeError as e:
    assert "4-bit product" in str(e)
else:
    raise AssertionError("not reported")
ops.check_device_status()
print("reported")
"""


def test_a_capture_that_comes_first_has_a_status_word():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "reported" in done.stdout, done.stderr[-2000:]
