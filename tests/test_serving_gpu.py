"""The serving operators against plain 64-bit restatements, at the sizes, masks and layouts where they can go wrong."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from intent_ir_b200.errors import B200LoweringError, B200RuntimeError  # noqa: E402

from . import serving_reference as ref  # noqa: E402

E4M3, I8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def ops():
    from intent_ir_b200 import ops as module
    return module


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _placed(t):
    """On the GPU with the strides and the storage offset that it has."""
    last = t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
    return torch.as_strided(torch.as_strided(t, (last,), (1,), 0).cuda(), t.shape, t.stride(), t.storage_offset())


# ---- rms-norm ---------------------------------------------------------------------------------------

def _check_norm(ops, x, w, residual, eps, out_dtype, group, **more):
    y, scale, h = ops.rmsnorm(_placed(x), None if w is None else _placed(w), residual=None if residual is None else _placed(residual), eps=eps,
                              out_dtype=out_dtype, group=group, **more)
    want_h, want = ref.rmsnorm(x, w, residual, eps)
    cols = x.shape[-1]
    # squares summed in f32: at most cols / 8 additions deep in any order used here, halved by the root, and ten more roundings
    slack = (cols / 16 + 16) * 2.0**-24
    if residual is None:
        assert h is None
    else:
        out = ref.half_step(x.dtype)
        assert ((h.cpu().double() - want_h).abs() <= want_h.abs() * out + 2.0**-24 * (x.double().abs() + residual.double().abs())).all()
    assert y.shape == x.shape
    if scale is None:
        assert y.dtype == x.dtype
        off = (y.cpu().double() - want).abs()
        assert (off <= want.abs() * (slack + ref.half_step(x.dtype)) + 2.0**-25 * (x.dtype == F16) + 1e-40).all(), off.max()
    else:
        assert scale.shape == x.shape[:-1] + ((-(-cols // group) if group else 1),)
        ref.check_held(y.cpu(), scale.cpu(), want, group, slack)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (5, 64), (2, 100), (17, 256), (4, 1000), (3, 1024), (2, 4096), (5, 5001), (2, 8192), (3, 8200), (1, 16384), (2, 40000)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rmsnorm_same_type(ops, rows, cols, dtype):
    g = _gen(rows * 100003 + cols)
    x, r, w = (torch.randn(s, generator=g).to(dtype) for s in ((rows, cols), (rows, cols), (cols,)))
    _check_norm(ops, x, w, r, 1e-5, None, 0)
    _check_norm(ops, x, None, None, 1e-6, None, 0)
    _check_norm(ops, x, w.float(), None, 1e-6, None, 0)


@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 33), (7, 40), (2, 248), (5, 256), (4, 1000), (3, 1024), (33, 4096), (2, 5003), (3, 8192), (2, 16640), (1, 36864)])
@pytest.mark.parametrize("out,group", [(E4M3, 0), (E4M3, 32), (E4M3, 128), (I8, 0), (I8, 64), (I8, 256)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rmsnorm_eight_bits(ops, rows, cols, out, group, dtype):
    g = _gen(rows * 7 + cols)
    x, r, w = (torch.randn(s, generator=g).to(dtype) for s in ((rows, cols), (rows, cols), (cols,)))
    x[0, cols // 2] = 60.0  # an outlier
    _check_norm(ops, x, w, r, 1e-6, out, group)
    _check_norm(ops, x, w, None, 1e-6, out, group)


def test_rmsnorm_zero_rows_tiny_and_huge_values(ops):
    x = torch.zeros(6, 512)
    x[1] = 1e-30
    x[2] = torch.randn(512, generator=_gen(1)) * 1e25  # squares beyond f32
    x[3, 5] = 3e38
    x[4] = torch.randn(512, generator=_gen(2)) * 1e18
    x[5] = torch.randn(512, generator=_gen(3))
    for out, group in ((None, 0), (E4M3, 0), (E4M3, 64), (I8, 0), (I8, 128)):
        _check_norm(ops, x, None, None, 1e-6, out, group)
        _check_norm(ops, x.to(BF16), None, None, 1e-6, out, group)
    y, scale, _ = ops.rmsnorm(x[:1].cuda(), out_dtype=I8)
    assert (y == 0).all() and (scale == 0).all()


@pytest.mark.parametrize("cols", [200, 250, 256, 512, 501, 1024, 1000, 2048, 1537, 4096, 2050])
@pytest.mark.parametrize("out_dtype,group", [(None, 0), (E4M3, 0), (E4M3, 64), (I8, 256)])
def test_rmsnorm_more_rows_than_the_gpu_takes_at_once(ops, cols, out_dtype, group):
    g = _gen(cols)
    x, r = (torch.randn(601, cols, generator=g).to(BF16) for _ in range(2))
    _check_norm(ops, x, torch.rand(cols, generator=g), r, 1e-5, out_dtype, group)
    _check_norm(ops, x.float(), None, None, 1e-5, out_dtype, group)
    x[7] *= 2.0**70  # squares beyond f32: the row is summed again
    _check_norm(ops, x, None, r, 1e-5, out_dtype, group)


@pytest.mark.parametrize("cols", [2, 6, 250, 1002, 3084, 5002, 10002])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift", [0, 1, 2])
def test_rmsnorm_rows_that_begin_on_pairs(ops, cols, dtype, shift):
    """Even widths; rows, residuals and weights that begin where pairs do, or `shift` elements later."""
    g = _gen(cols + shift)
    a, b = (torch.randn(5, cols + 2, generator=g).to(dtype) for _ in range(2))
    w = torch.randn(cols + 2, generator=g)
    for out_dtype in (None, E4M3, I8):
        _check_norm(ops, a[:, shift:shift + cols], None, b[:, :cols], 1e-5, out_dtype, 0)
        _check_norm(ops, a[:, :cols], w.to(dtype)[:cols], b[:, shift:shift + cols], 1e-5, out_dtype, 0)
        _check_norm(ops, a[:, :cols], w[shift:shift + cols], None, 1e-5, out_dtype, 0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rmsnorm_non_finite_rows_stand_for_nan_and_touch_no_other_row(ops, bad):
    x = torch.randn(4, 640, generator=_gen(5))
    x[2, 77] = bad
    y, _, _ = ops.rmsnorm(x.cuda())
    _, want = ref.rmsnorm(x, None, None, 1e-6)
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
    for out in (E4M3, I8):
        for group in (0, 64):
            y, scale, _ = ops.rmsnorm(x.cuda(), out_dtype=out, group=group)
            value = y.cpu().double() * ref.spread_scale(scale.cpu().double(), 640, group)
            assert torch.isnan(value[2][torch.isnan(want[2])]).all() and torch.isfinite(value[[0, 1, 3]]).all()


def test_rmsnorm_strided_rows_in_place_and_leading_axes(ops):
    wide = torch.randn(9, 3 * 512 + 8, generator=_gen(7)).to(BF16)
    r = torch.randn(9, 512, generator=_gen(8)).to(BF16)
    for at in (0, 512, 515):  # the last one is not on a 16-byte boundary
        x = wide.cuda()[:, at:at + 512]
        want, _, h = ops.rmsnorm(x.contiguous(), residual=r.cuda(), out_dtype=E4M3)
        res = r.cuda()
        got, _, h2 = ops.rmsnorm(x, residual=res, out_dtype=E4M3, residual_out=res)
        assert h2 is res and torch.equal(h2, h) and torch.equal(got.view(torch.uint8), want.view(torch.uint8))
        box = wide.cuda()
        _, _, h3 = ops.rmsnorm(box[:, at:at + 512], residual=r.cuda(), residual_out=box[:, at:at + 512])
        assert torch.equal(h3, h)
        untouched = torch.ones(box.shape[1], dtype=torch.bool)
        untouched[at:at + 512] = False
        assert torch.equal(box.cpu()[:, untouched], wide[:, untouched])
    x = torch.randn(2, 3, 5, 96, generator=_gen(9))
    _check_norm(ops, x, None, x * 2, 1e-6, I8, 32)
    y, scale, h = ops.rmsnorm(torch.empty(0, 64, device="cuda"), out_dtype=I8)
    assert y.shape == (0, 64) and scale.shape == (0, 1) and h is None


def test_rmsnorm_refusals(ops):
    x = torch.randn(4, 64, device="cuda")
    for bad in (dict(out_dtype=torch.uint8), dict(out_dtype=BF16), dict(out_dtype=I8, group=48), dict(out_dtype=I8, group=-32), dict(group=32)):
        with pytest.raises(B200LoweringError):
            ops.rmsnorm(x, **bad)
    with pytest.raises(B200LoweringError):
        ops.rmsnorm(x.double())
    with pytest.raises(B200LoweringError):
        ops.rmsnorm(x, torch.ones(64, device="cuda", dtype=torch.int8))
    with pytest.raises(B200LoweringError):
        ops.rmsnorm(x, torch.ones(64, device="cuda", dtype=BF16))
    for bad in (dict(w=torch.ones(63, device="cuda")), dict(w=torch.ones(64)), dict(residual=x[:3]), dict(residual=x.half()), dict(residual_out=x),
                dict(residual=x, residual_out=x[:2])):
        with pytest.raises(B200RuntimeError):
            ops.rmsnorm(x, **bad)
    with pytest.raises(B200RuntimeError):
        ops.rmsnorm(x.t())
    with pytest.raises(B200RuntimeError):
        ops.rmsnorm(x.cpu())


def test_rmsnorm_beyond_two_billion_elements(ops):
    rows, cols = 140000, 16384
    x = torch.empty(rows, cols, dtype=BF16, device="cuda")
    x[:] = torch.randn(cols, device="cuda").to(BF16)
    x[-3:] = torch.randn(3, cols, device="cuda").to(BF16)
    y, scale, _ = ops.rmsnorm(x, out_dtype=E4M3, group=128)
    _, want = ref.rmsnorm(x[-4:].cpu(), None, None, 1e-6)
    ref.check_held(y[-4:].cpu(), scale[-4:].cpu(), want, 128, (cols / 16 + 16) * 2.0**-24)


# ---- products with 4-bit weights --------------------------------------------------------------------

def _w4_case(m, n, k, dtype, group, zeros, bias, x_groups, scale_dtype, seed=0, out_dtype=None):
    g = _gen(seed + m * 31 + n * 17 + k)
    groups = -(-k // group)
    out_dtype = out_dtype or (BF16 if dtype in (E4M3, I8) else dtype)
    d = {"q": torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8), "group": group,
         "scales": (torch.rand(n, groups, generator=g) * 0.02 + 0.001).to(scale_dtype),
         "zeros": torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None,
         "bias": torch.randn(n, generator=g).to(out_dtype) if bias else None, "x_scale": None}
    x = torch.randn(m, k, generator=g)
    if dtype in (E4M3, I8):
        x = x * 30
        d["x"] = x.clamp(-127, 127).round().to(I8) if dtype == I8 else x.to(E4M3)
        d["x_scale"] = torch.rand(m, x_groups or 1 if x_groups == 1 else groups, generator=g) * 0.05 + 0.01
    else:
        d["x"] = x.to(dtype)
    return d, out_dtype


def _check_w4(ops, d, out_dtype):
    got = ops.w4_matmul(**{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in d.items()}, out_dtype=out_dtype)
    want, size = ref.w4_matmul(**d)
    assert got.dtype == out_dtype and got.shape == want.shape
    off = (got.cpu().double() - want).abs()
    bound = ref.w4_bound(want, size, d["x"].shape[-1], out_dtype)
    assert (off <= bound).all(), ((off / bound).max(), (off > bound).sum())
    return got


@pytest.mark.parametrize("m", [1, 2, 3, 8, 9, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (5, 64, 128), (16, 128, 64), (77, 160, 128), (130, 1056, 32), (300, 2080, 64), (1027, 512, 128), (256, 4096, 128)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_w4_sizes(ops, m, n, k, group, dtype):
    _check_w4(ops, *_w4_case(m, n, k, dtype, group, m % 2 == 0, n % 2 == 1, 0, dtype if m % 3 else F32))


@pytest.mark.parametrize("m", [1, 5, 8, 20, 64, 100])
@pytest.mark.parametrize("n,k,group", [(33, 32, 128), (64, 224, 64), (200, 1120, 32), (515, 2048, 128)])
@pytest.mark.parametrize("dtype", [E4M3, I8])
@pytest.mark.parametrize("x_groups", [1, 2])
def test_w4_eight_bit_activations(ops, m, n, k, group, dtype, x_groups):
    _check_w4(ops, *_w4_case(m, n, k, dtype, group, n % 2 == 0, True, x_groups, [F32, BF16, F16][m % 3], out_dtype=[BF16, F16, F32][n % 3]))


@pytest.mark.parametrize("m", [1, 4, 12, 40])
def test_w4_every_nibble_and_position(ops, m):
    """x one-hot: every weight comes back exactly."""
    n, k, group = 32, 256, 32
    d, _ = _w4_case(m, n, k, F16, group, True, False, 0, F32)
    d["scales"] = torch.ones_like(d["scales"])
    w = ref.w4_weights(d["q"], d["scales"], d["zeros"], group)
    for at in range(0, k, m):
        x = torch.zeros(m, k, dtype=F16)
        for i in range(min(m, k - at)):
            x[i, at + i] = 1.0
        d["x"] = x
        got = ops.w4_matmul(**{a: b.cuda() if isinstance(b, torch.Tensor) else b for a, b in d.items()})
        assert torch.equal(got[:k - at].cpu().double(), w[:, at:at + m].t())


def test_w4_strides_axes_large_values_and_empty(ops):
    d, out = _w4_case(6, 100, 256, BF16, 64, False, False, 0, BF16)
    want = _check_w4(ops, d, out)
    wide = torch.zeros(6, 300, dtype=BF16)
    for at in (0, 8, 13):
        wide[:, at:at + 256] = d["x"]
        got = ops.w4_matmul(wide.cuda()[:, at:at + 256], d["q"].cuda(), d["scales"].cuda(), group=64)
        assert torch.equal(got, want)
    got = ops.w4_matmul(d["x"].cuda().view(2, 3, 256), d["q"].cuda(), d["scales"].cuda(), group=64)
    assert got.shape == (2, 3, 100) and torch.equal(got.view(6, 100), want)
    d["x"] = (d["x"].float() * 1e30).to(BF16)  # far beyond f16
    _check_w4(ops, d, out)
    d["x"][2, 7], d["x"][4, 9] = float("inf"), float("nan")
    got = ops.w4_matmul(d["x"].cuda(), d["q"].cuda(), d["scales"].cuda(), group=64).cpu()
    assert not torch.isfinite(got[2]).any() or (ref.unpack(d["q"])[:, 7] == 8).any()
    assert torch.isnan(got[4]).all() and torch.isfinite(got[[0, 1, 3, 5]]).all()
    assert ops.w4_matmul(torch.empty(0, 256, dtype=BF16, device="cuda"), d["q"].cuda(), d["scales"].cuda(), group=64).shape == (0, 100)
    bias = torch.randn(7, device="cuda", dtype=BF16)
    empty = ops.w4_matmul(torch.empty(2, 0, dtype=BF16, device="cuda"), torch.empty(7, 0, dtype=torch.uint8, device="cuda"),
                          torch.empty(7, 0, dtype=BF16, device="cuda"), bias=bias)
    assert torch.equal(empty, bias.expand(2, 7))


@pytest.mark.parametrize("m", [1, 12, 40])
def test_w4_scales_and_zero_points_off_their_boundaries(ops, m):
    """Groups that fill their blocks of eight or not, in arrays that begin anywhere."""
    for k, group in ((2048, 128), (2048, 32), (1056, 32), (1152, 128)):
        for scale_dtype in (BF16, F32):
            d, out = _w4_case(m, 150, k, F16, group, True, True, 0, scale_dtype)
            want = _check_w4(ops, d, out)
            e = {n: v.cuda() if isinstance(v, torch.Tensor) else v for n, v in d.items()}
            for name in ("scales", "zeros", "bias"):
                box = torch.empty(e[name].numel() + 3, dtype=e[name].dtype, device="cuda")
                for off in (1, 3):
                    view = box[off:off + e[name].numel()].view(e[name].shape)
                    view.copy_(e[name])
                    assert torch.equal(ops.w4_matmul(**{**e, name: view}, out_dtype=out), want), (k, group, name, off)


@pytest.mark.parametrize("m", [9, 16])
def test_w4_larger_matrices_with_a_few_rows(ops, m):
    d, out = _w4_case(m, 8200, 8192, BF16, 128, m == 9, False, 0, BF16)
    _check_w4(ops, d, out)


@pytest.mark.parametrize("m", [1, 20])
def test_w4_weights_beyond_two_gigabytes(ops, m):
    n, k, group = 66000, 65536, 128
    q = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    scales = (torch.rand(n, k // group, device="cuda") * 0.01).to(BF16)
    x = torch.randn(m, k, device="cuda").to(BF16)
    got = ops.w4_matmul(x, q, scales, group=group)
    for at in (0, 65520, n - 40):
        part = {"x": x.cpu(), "q": q[at:at + 40].cpu(), "scales": scales[at:at + 40].cpu(), "zeros": None, "bias": None, "x_scale": None, "group": group}
        want, size = ref.w4_matmul(**part)
        assert ((got[:, at:at + 40].cpu().double() - want).abs() <= ref.w4_bound(want, size, k, BF16)).all()


def test_w4_refusals(ops):
    d, _ = _w4_case(4, 64, 256, BF16, 64, True, True, 0, BF16)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in d.items()}
    ops.w4_matmul(**d)
    for bad in (dict(group=48), dict(group=256), dict(q=d["q"][0]), dict(x=d["x"].float()), dict(x=d["x"][:, :200]), dict(out_dtype=torch.int8), dict(out_dtype=I8, bias=None),
                dict(scales=d["scales"].double())):
        with pytest.raises(B200LoweringError):
            ops.w4_matmul(**{**d, **bad})
    for bad in (dict(q=d["q"][:, :100]), dict(q=d["q"].view(torch.int8)), dict(scales=d["scales"][:, :3]), dict(zeros=d["zeros"][:10]), dict(zeros=d["scales"]),
                dict(bias=d["bias"][:3]), dict(bias=d["bias"].float()), dict(x_scale=torch.ones(4, 1, device="cuda")), dict(x=d["x"].cpu()), dict(q=d["q"].cpu()),
                dict(x=d["x"].to(I8)), dict(x=d["x"].to(I8), x_scale=torch.ones(4, 2, device="cuda")), dict(x=d["x"].to(I8), x_scale=torch.ones(4, 1, device="cuda", dtype=BF16)),
                dict(q=d["q"].t().contiguous().t())):
        with pytest.raises(B200RuntimeError):
            ops.w4_matmul(**{**d, **bad})
    odd = torch.empty(64 * 128 + 1, dtype=torch.uint8, device="cuda")[1:].view(64, 128)
    with pytest.raises(B200RuntimeError):
        ops.w4_matmul(**{**d, "q": odd})


# ---- the 8-bit paged cache --------------------------------------------------------------------------

def _paged(seed, news, lens, heads, dim, block, dtype, held, slack_pages=3, table_blocks=None, spread=1.0):
    """Random caches, a shuffled table, new keys, values and queries' offsets; the slots that no sequence has written hold the type's worst byte."""
    g = _gen(seed)
    per = [max(0, -(-max(x, 0) // block)) for x in lens]
    pages = sum(per) + slack_pages
    order = torch.randperm(pages, generator=g).to(torch.int32)
    width = table_blocks if table_blocks is not None else max(per + [1]) + 1
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    at = 0
    for b, count in enumerate(per):
        table[b, :min(count, width)] = order[at:at + count][:width]
        at += count
    d = {"block_table": table, "seq_lens": torch.tensor(lens, dtype=torch.int32),
         "cu_new": torch.tensor([0] + news).cumsum(0).to(torch.int32)}
    total = sum(news)
    for name in ("k", "v"):
        d[name] = (torch.randn(total, heads, dim, generator=g) * spread).to(dtype)
        scale = torch.rand(pages, heads, generator=g) * 0.02 + 0.001
        cache = torch.empty(pages, heads, block, dim, dtype=torch.uint8)
        if held == I8:
            cache = torch.randint(-127, 128, cache.shape, generator=g).to(I8)
            worst = torch.full_like(cache, -128)
        else:
            cache = (torch.randn(cache.shape, generator=g) * 100).clamp(-448, 448).to(E4M3)
            worst = torch.full(cache.shape, 0x7F, dtype=torch.uint8).view(E4M3)
        used = torch.zeros(pages, block, dtype=torch.bool)
        for b, x in enumerate(lens):
            for j in range(min(per[b], width)):
                used[int(table[b, j]), :max(0, min(block, x - j * block))] = True
        bits = torch.where(used[:, None, :, None], cache.view(torch.uint8), worst.view(torch.uint8))
        d[name + "_cache"], d[name + "_scale"] = bits.view(held), scale
    return d


def _on_gpu(t):
    """On the GPU with the strides it has."""
    return t.cuda() if t.is_contiguous() else _placed(t)


def _cuda(d):
    return {k: _on_gpu(v) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


CACHE = ("k_cache", "v_cache", "k_scale", "v_scale")


def _check_append(ops, d, uniform=False):
    dev = _cuda(d)
    ops.kv8_append(dev["k"], dev["v"], *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"], cu_new=None if uniform else dev["cu_new"])
    want = {c: d[c].clone() for c in CACHE}
    ref.append(d["k"], d["v"], *(want[c] for c in CACHE), d["block_table"], d["seq_lens"], d["cu_new"])
    for c in CACHE:
        got = dev[c].cpu()
        if c.endswith("cache"):
            a, b = got.view(torch.uint8), want[c].view(torch.uint8)
            nan = (a & 0x7F == 0x7F) & (b & 0x7F == 0x7F) if got.dtype == E4M3 else torch.zeros_like(a, dtype=torch.bool)
            assert ((a == b) | nan).all(), (c, (a != b).nonzero()[:5])
        else:
            assert torch.equal(got.nan_to_num(nan=-1.0), want[c].nan_to_num(nan=-1.0)), c
    return dev


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,dim,block,dtype", [(1, 64, 16, F16), (3, 128, 16, BF16), (2, 128, 48, F16), (4, 64, 64, BF16), (1, 128, 1024, BF16)])
def test_append_matches_the_definition_bit_for_bit(ops, held, heads, dim, block, dtype):
    _check_append(ops, _paged(1, [1, 1, 1, 1], [1, 16, 17, 1025], heads, dim, block, dtype, held), uniform=True)
    _check_append(ops, _paged(2, [3, 3], [40, 3], heads, dim, block, dtype, held), uniform=True)
    _check_append(ops, _paged(3, [5, 1, 0, 100, 33], [5, 90, 12, 130, 64], heads, dim, block, dtype, held))
    _check_append(ops, _paged(4, [1, 20], [50, 31], heads, dim, block, dtype, held, spread=1e-3))  # nothing grows
    _check_append(ops, _paged(5, [1, 20], [50, 31], heads, dim, block, dtype, held, spread=300.0))  # everything grows


@pytest.mark.parametrize("held", [E4M3, I8])
def test_append_one_token_at_a_time_equals_its_definition_and_ends_full(ops, held):
    d = _paged(9, [1, 1], [1, 1], 2, 64, 16, BF16, held, slack_pages=6)
    d["block_table"] = torch.tensor([[4, 2, 0], [1, 3, 5]], dtype=torch.int32)
    dev = _cuda(d)
    for n in range(1, 40):
        d["k"], d["v"] = (torch.randn(2, 2, 64, generator=_gen(n + i)).to(BF16) * n for i in (0, 1000))
        d["seq_lens"] = torch.tensor([n, n], dtype=torch.int32)
        ops.kv8_append(d["k"].cuda(), d["v"].cuda(), *(dev[c] for c in CACHE), dev["block_table"], d["seq_lens"].cuda())
        ref.append(d["k"], d["v"], *(d[c] for c in CACHE), d["block_table"], d["seq_lens"], d["cu_new"])
    for c in CACHE:
        assert torch.equal(dev[c].cpu().view(torch.uint8), d[c].view(torch.uint8))


@pytest.mark.parametrize("held", [E4M3, I8])
def test_append_leaves_bad_pages_and_tokens_outside_alone(ops, held):
    d = _paged(11, [4, 20, 2, 3], [30, 40, 1, 100], 2, 64, 16, BF16, held, table_blocks=3)  # the third has fewer tokens than new ones, the fourth runs out of table
    d["block_table"][1, 1], d["block_table"][1, 2] = 10**9, -1
    d["cu_new"] = torch.tensor([0, 4, 24, 26, 29], dtype=torch.int32)
    d["k"], d["v"] = (torch.cat((d[x], d[x][:5])) for x in ("k", "v"))  # five tokens behind the last sequence
    _check_append(ops, d)


@pytest.mark.parametrize("held", [E4M3, I8])
def test_append_zeros_and_non_finite_values(ops, held):
    d = _paged(12, [3, 3, 3], [20, 3, 19], 2, 64, 16, F16, held)
    d["k"][:3] = 0
    d["v"][3:6] = 0  # a block of zeros alone
    d["k"][7, 1, 5] = float("nan")
    d["v"][6, 0, 9] = float("inf")
    dev = _cuda(d)
    ops.kv8_append(dev["k"], dev["v"], *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"], cu_new=dev["cu_new"])
    page = int(d["block_table"][1, 0])
    assert (dev["v_cache"][page, :, :3].float() == 0).all() and (dev["v_scale"][page] == 0).all()
    page = int(d["block_table"][2, 1])
    for name, head, other in (("k", 1, 0), ("v", 0, 1)):
        value = dev[name + "_cache"][page].float() * dev[name + "_scale"][page][:, None, None]
        assert torch.isnan(value[head, :3]).all() and torch.isfinite(value[other, :3]).all()
    for c in CACHE:
        d[c] = dev[c].cpu()
    q = torch.randn(9, 2, 64, generator=_gen(1)).to(F16)
    o = ops.attention_kv8(q.cuda(), *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"], cu_new=dev["cu_new"]).cpu()
    assert torch.isfinite(o[:6]).all()
    assert torch.isnan(o[6:]).all()


@pytest.mark.parametrize("held", [E4M3, I8])
def test_append_and_attention_in_a_cache_beyond_two_billion_values(ops, held):
    d = _paged(14, [3, 40], [70, 300], 8, 128, 16, BF16, held)
    q = torch.randn(43, 8, 128, generator=_gen(2)).to(BF16)
    small = _cuda(d)
    pages, used = 140000, d["k_cache"].shape[0]
    big = dict(small, block_table=torch.where(small["block_table"] >= 0, small["block_table"] + (pages - used), small["block_table"]))
    for c in CACHE:
        big[c] = torch.zeros((pages,) + tuple(small[c].shape[1:]), dtype=small[c].dtype, device="cuda")
        big[c][pages - used:].view(torch.uint8).copy_(small[c].view(torch.uint8))
    out = []
    for s in (small, big):
        args = [s[c] for c in CACHE] + [s["block_table"], s["seq_lens"]]
        ops.kv8_append(s["k"], s["v"], *args, cu_new=s["cu_new"])
        out.append(ops.attention_kv8(q.cuda(), *args, cu_new=s["cu_new"]))
    assert torch.equal(*out) and torch.isfinite(out[0]).all()
    for c in CACHE:
        assert torch.equal(big[c][pages - used:].view(torch.uint8), small[c].view(torch.uint8))
        assert not big[c][:pages - used].view(torch.uint8).any()


@pytest.mark.parametrize("held", [E4M3, I8])
def test_append_a_padded_batch(ops, held):
    """Sequences of length 0 with a place among the new tokens: nothing is written for them."""
    d = _paged(15, [1] * 5, [40, 0, 17, 0, 0], 2, 64, 16, BF16, held)
    _check_append(ops, d, uniform=True)
    _check_attention(ops, {**d}, 4, uniform=True)


def test_append_strided_inputs(ops):
    d = _paged(13, [2, 7], [20, 39], 3, 64, 16, BF16, E4M3)
    fused = torch.randn(9, 5 * 3, 64, generator=_gen(3)).to(BF16)
    d["k"], d["v"] = fused[:, 3:6], fused[:, 9:12]
    _check_append(ops, d)
    swapped = fused[:, :6].transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    d["k"], d["v"] = swapped[:, :3], swapped[:, 3:]
    _check_append(ops, d)


# ---- attention --------------------------------------------------------------------------------------

def _check_attention(ops, d, q_heads, uniform=False, scale=None, window=0, seed=0, q=None):
    heads, dim = d["k_cache"].shape[1], d["k_cache"].shape[3]
    if q is None:
        q = torch.randn(d["k"].shape[0], q_heads, dim, generator=_gen(seed + 77)).to(d["k"].dtype) * 1.5
    out = torch.full(q.shape, 7.0, dtype=q.dtype).cuda()
    dev = _cuda(d)
    got, lse = ops.attention_kv8(_on_gpu(q), *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"], cu_new=None if uniform else dev["cu_new"], scale=scale,
                                 window=window, return_lse=True, out=out)
    assert got is out
    want, want_lse, bound, lse_bound = ref.attention(q, *(d[c] for c in CACHE), d["block_table"], d["seq_lens"], d["cu_new"],
                                                     dim ** -0.5 if scale is None else scale, window)
    covered = torch.zeros(q.shape[0], dtype=torch.bool)
    covered[int(d["cu_new"][0]):int(d["cu_new"][-1])] = True
    got, lse = got.cpu().double(), lse.cpu().double()
    assert (got[~covered] == 7.0).all()
    got, lse, want, want_lse, bound, lse_bound = (x[covered] for x in (got, lse, want, want_lse, bound, lse_bound))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    ok = ((got - want).abs() <= bound) | torch.isnan(want)
    assert ok.all(), ((got - want).abs() / bound).nan_to_num().max()
    ok = ((lse - want_lse).abs() <= lse_bound) | torch.isnan(want_lse) | (lse == want_lse)
    assert ok.all(), (lse - want_lse).abs().nan_to_num().max()


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim,block,dtype", [(1, 1, 64, 16, F16), (2, 3, 128, 16, BF16), (3, 8, 128, 48, F16), (2, 16, 64, 64, BF16), (1, 9, 128, 32, BF16), (2, 32, 128, 1024, F16)])
def test_attention_single_tokens(ops, held, heads, group, dim, block, dtype):
    lens = [1, 15, 16, 17, 31, 33, 64, 127, 128, 129, 500, 1030]
    _check_attention(ops, _paged(21, [1] * len(lens), lens, heads, dim, block, dtype, held), heads * group, uniform=True)


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("heads,group,dim,block,dtype", [(2, 1, 64, 16, F16), (2, 4, 128, 16, BF16), (1, 7, 128, 64, F16)])
@pytest.mark.parametrize("window", [0, 1, 40, 257])
def test_attention_several_tokens_and_windows(ops, held, heads, group, dim, block, dtype, window):
    _check_attention(ops, _paged(22, [4, 1, 0, 9, 70], [4, 300, 12, 9, 400], heads, dim, block, dtype, held), heads * group, window=window)
    _check_attention(ops, _paged(23, [3, 3, 3], [3, 100, 260], heads, dim, block, dtype, held), heads * group, uniform=True, window=window)


@pytest.mark.parametrize("held", [E4M3, I8])
def test_attention_long_sequences_beside_short_ones(ops, held):
    _check_attention(ops, _paged(24, [1] * 5, [20000, 3, 700, 1, 9001], 2, 128, 32, BF16, held), 8, uniform=True)
    _check_attention(ops, _paged(25, [2, 1, 2], [30001, 1, 77], 1, 64, 16, F16, held), 4)


@pytest.mark.parametrize("held", [E4M3, I8])
def test_attention_many_sequences(ops, held):
    """More sequences than a CTA has threads, and pages that several of them share."""
    lens = [(i * 37) % 200 for i in range(300)]
    d = _paged(31, [1] * 300, lens, 1, 64, 16, BF16, held)
    _check_attention(ops, d, 4, uniform=True)
    news = [i % 3 for i in range(290)]
    d = _paged(32, news, [max(n, x) for n, x in zip(news, lens)], 2, 64, 16, F16, held)
    d["block_table"][5:40] = d["block_table"][4]  # read by all: nobody appends here
    d["seq_lens"][5:40] = d["seq_lens"][4]
    _check_attention(ops, d, 2, window=50)


@pytest.mark.parametrize("held", [E4M3, I8])
def test_attention_empty_rows_padding_and_bad_pages(ops, held):
    d = _paged(26, [2, 3, 1, 2, 4, 1], [0, 1, 50, 300, 90, 20], 2, 64, 16, BF16, held, table_blocks=6)  # none, fewer than new, .., longer than the table
    d["block_table"][4, 2] = 1 << 30
    d["block_table"][5, 0] = -5
    d["k"] = torch.cat((d["k"], d["k"][:4]))  # four rows behind the last sequence
    _check_attention(ops, d, 4)
    _check_attention(ops, d, 4, window=20)
    d["seq_lens"][0] = -3
    _check_attention(ops, d, 4)


def test_attention_extreme_scores(ops):
    d = _paged(27, [1, 1, 2], [200, 333, 64], 2, 64, 16, F16, E4M3)
    for factor, scale in ((1.0, 0.0), (1.0, -0.3), (100.0, 0.125), (6e4, 1e-4), (1e-7, 1e5)):
        q = (torch.randn(4, 4, 64, generator=_gen(3)) * factor).clamp(-65000, 65000).to(F16)
        _check_attention(ops, d, 4, scale=scale, q=q)
    d = _paged(28, [1, 1], [200, 333], 2, 128, 16, BF16, E4M3)
    q = (torch.randn(2, 2, 128, generator=_gen(4)) * 1e20).to(BF16)  # beyond f16
    _check_attention(ops, d, 2, scale=1e-21, q=q)
    for name in ("k_scale", "v_scale"):
        d[name] *= torch.logspace(-6, 6, d[name].shape[0])[torch.randperm(d[name].shape[0], generator=_gen(5))][:, None]
    _check_attention(ops, d, 2, scale=1e-3)


def test_attention_non_finite_queries_and_scales_stay_in_their_rows(ops):
    d = _paged(29, [1, 1, 1], [40, 300, 90], 2, 64, 16, BF16, I8)
    q = torch.randn(3, 4, 64, generator=_gen(6)).to(BF16)
    q[0, 1, 3] = float("nan")
    q[2, 2, 60] = float("inf")
    d["v_scale"][int(d["block_table"][1, 4]), 1] = float("nan")
    dev = _cuda(d)
    o = ops.attention_kv8(q.cuda(), *(dev[c] for c in CACHE), dev["block_table"], dev["seq_lens"]).cpu()
    bad = torch.isnan(o).all(-1)
    want = torch.zeros(3, 4, dtype=torch.bool)
    want[0, 1] = want[2, 2] = want[1, 2] = want[1, 3] = True
    assert torch.equal(bad, want) and torch.isfinite(o[~want]).all()


def test_attention_strides_refusals_and_empty(ops):
    d = _paged(30, [1, 1, 1], [40, 300, 90], 2, 64, 16, BF16, E4M3)
    fused = torch.randn(3, 9, 64, generator=_gen(8)).to(BF16)
    _check_attention(ops, d, 4, q=fused[:, 2:6])
    dev = _cuda(d)
    args = [dev[c] for c in CACHE] + [dev["block_table"], dev["seq_lens"]]
    q = fused[:, :4].cuda()
    assert ops.attention_kv8(q[:0], *args, cu_new=torch.zeros(4, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    for bad in (dict(q=q.float()), dict(k_cache=dev["k_cache"].view(torch.uint8), v_cache=dev["v_cache"].view(torch.uint8))):
        names = dict(zip(("q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seq_lens"), [q] + args))
        with pytest.raises(B200LoweringError):
            ops.attention_kv8(**{**names, **bad})
    for bad in (dict(q=q[:, :3]), dict(q=q[:2]), dict(q=q[:, :, :32]), dict(q=q.cpu()), dict(v_cache=dev["v_cache"][:2]), dict(k_scale=dev["k_scale"].double()),
                dict(block_table=dev["block_table"].long()), dict(block_table=dev["block_table"][:2]), dict(seq_lens=dev["seq_lens"].cpu()), dict(window=-1),
                dict(cu_new=torch.zeros(3, dtype=torch.int32, device="cuda")), dict(out=torch.empty_like(q)[:2]), dict(out=torch.empty(3, 4, 64)),
                dict(k_scale=None)):
        with pytest.raises(B200RuntimeError):
            ops.attention_kv8(**{**names, **bad})
    with pytest.raises(B200RuntimeError):
        ops.kv8_append(dev["k"], dev["v"][:2], *args)
    with pytest.raises(B200RuntimeError):
        ops.kv8_append(dev["k"][:, :1], dev["v"][:, :1], *args)


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (64, BF16), (128, F16), (128, BF16)])
def test_attention_units_of_twenty_four_rows(ops, held, dim, dtype):
    """Taken where a table has room for more tiles than the GPU takes at once: a cluster to a unit, the even split, ragged sequences."""
    for room, window in ((400, 0), (1200, 0), (1200, 100)):
        d = _paged(60, [5, 5, 5], [700, 3, 131], 2, dim, 16, dtype, held, table_blocks=room)
        if held == E4M3:  # the last new token's value is NaN: only its own rows see it
            page, slot = int(d["block_table"][0, 699 // 16]), 699 % 16
            d["v_cache"].view(torch.uint8)[page, 1, slot, 3] = 0x7F
        _check_attention(ops, d, 8, uniform=True, window=window)  # 20 rows
        _check_attention(ops, d, 16, uniform=True, window=window)  # 40 rows: the second unit has 16
    d = _paged(61, [20, 9, 14, 1], [600, 9, 3, 77], 2, dim, 16, dtype, held, table_blocks=600)
    _check_attention(ops, d, 10)  # 100 rows, 45, 70, 5
    _check_attention(ops, d, 10, window=33)


def test_heads_without_width_are_refused(ops):
    d = _cuda(_paged(31, [1, 1], [5, 20], 2, 64, 16, BF16, E4M3))
    caches = [d["k_cache"][..., :0].contiguous(), d["v_cache"][..., :0].contiguous(), d["k_scale"], d["v_scale"], d["block_table"], d["seq_lens"]]
    with pytest.raises(B200LoweringError):
        ops.attention_kv8(d["k"][..., :0], *caches)
    with pytest.raises(B200LoweringError):
        ops.kv8_append(d["k"][..., :0], d["v"][..., :0], *caches)


# ---- a run of them together -------------------------------------------------------------------------

def _layer(ops, s, held, out8):
    """One serving step: norm -> 4-bit projection to q, k, v -> append -> attention -> 4-bit projection -> norm with the residual."""
    y, ys, _ = ops.rmsnorm(s["x"], s["w1"], out_dtype=out8, group=0)
    qkv = ops.w4_matmul(y, s["q1"], s["s1"], zeros=s["z1"], x_scale=ys, group=64, out_dtype=BF16).view(-1, 4 + 2 + 2, 64)
    ops.kv8_append(qkv[:, 4:6], qkv[:, 6:8], *(s[c] for c in CACHE), s["block_table"], s["seq_lens"], cu_new=s["cu_new"])
    o = ops.attention_kv8(qkv[:, :4], *(s[c] for c in CACHE), s["block_table"], s["seq_lens"], cu_new=s["cu_new"])
    back = ops.w4_matmul(o.view(-1, 256), s["q2"], s["s2"], group=128)
    return ops.rmsnorm(back, s["w2"], residual=s["x"], out_dtype=out8, group=128)


def _layer_inputs(held):
    d = _paged(41, [1, 3, 1, 6], [70, 3, 16, 200], 2, 64, 16, BF16, held)
    g = _gen(42)
    d.update(x=torch.randn(11, 512, generator=g).to(BF16), w1=torch.rand(512, generator=g).to(BF16), w2=torch.rand(512, generator=g).to(BF16),
             q1=torch.randint(0, 256, (512, 256), generator=g, dtype=torch.uint8), s1=(torch.rand(512, 8, generator=g) * 0.02).to(BF16),
             z1=torch.randint(6, 10, (512, 8), generator=g, dtype=torch.uint8),
             q2=torch.randint(0, 256, (512, 128), generator=g, dtype=torch.uint8), s2=(torch.rand(512, 2, generator=g) * 0.02).to(BF16))
    return d


@pytest.mark.parametrize("held", [E4M3, I8])
@pytest.mark.parametrize("out8", [E4M3, I8])
def test_the_step_together(ops, held, out8):
    d = _layer_inputs(held)
    dev = _cuda(d)
    y, scale, h = _layer(ops, dev, held, out8)
    # the same in 64 bits, with the roundings between the operators
    _, n1 = ref.rmsnorm(d["x"], d["w1"], None, 1e-6)
    s = ref.group_max(n1, 0) / ref.TOP[out8]
    n1 = ref.hold((n1 / s).numpy(), out8).double() * s
    qkv = (n1 @ ref.w4_weights(d["q1"], d["s1"], d["z1"], 64).t()).to(BF16).view(-1, 8, 64)
    ref.append(qkv[:, 4:6], qkv[:, 6:8], *(d[c] for c in CACHE), d["block_table"], d["seq_lens"], d["cu_new"])
    o = ref.attention(qkv[:, :4], *(d[c] for c in CACHE), d["block_table"], d["seq_lens"], d["cu_new"], 0.125, 0)[0].to(BF16)
    back = (o.reshape(-1, 256).double() @ ref.w4_weights(d["q2"], d["s2"], None, 128).t()).to(BF16)
    want_h, want = ref.rmsnorm(back, d["w2"], d["x"], 1e-6)
    got = y.cpu().double() * ref.spread_scale(scale.cpu().double(), 512, 128)
    # three 8-bit roundings (2^-4 at most, of e4m3) and four of bf16 lie between the inputs and y; a rounding that falls to the other
    # side moves a value by one step, which the products average over hundreds of terms: the norm of the difference stays below one e4m3 step
    assert (got - want).norm() <= 2.0**-4 * want.norm()
    assert (h.cpu().double() - want_h).norm() <= 2.0**-6 * want_h.norm()
    again = _cuda(_layer_inputs(held))
    for a, b in zip(_layer(ops, again, held, out8), (y, scale, h)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # the same inputs, the same bits


def test_two_steps_at_once_on_two_streams(ops):
    want = [t.clone() for t in _layer(ops, _cuda(_layer_inputs(E4M3)), E4M3, I8)]
    states = [_cuda(_layer_inputs(E4M3)) for _ in range(8)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(states):
        with torch.cuda.stream(streams[i % 2]):
            got.append(_layer(ops, s, E4M3, I8))
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))


def test_the_step_on_another_stream_and_in_a_graph(ops):
    held, out8 = E4M3, E4M3
    want = [t.clone() for t in _layer(ops, _cuda(_layer_inputs(held)), held, out8)]
    side = torch.cuda.Stream()
    s = _cuda(_layer_inputs(held))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _layer(ops, s, held, out8)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):  # two graphs, each with its own scratch, replayed at once
        s = _cuda(_layer_inputs(held))
        fresh = {c: s[c].clone() for c in CACHE}
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _layer(ops, s, held, out8)
        graphs.append((g, out, s, fresh))
    for _ in range(3):
        for g, out, s, fresh in graphs:
            for c in CACHE:
                s[c].copy_(fresh[c])
            for t in out:
                t.view(torch.uint8).fill_(0xAB)
        torch.cuda.synchronize()
        other = torch.cuda.Stream()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for g, out, s, fresh in graphs:
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(out, want))
