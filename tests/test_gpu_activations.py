"""Packed activations on the GPU against the 64-bit checker."""

import io
import math

import pytest
import torch
from torch import nn

from helpers import assert_bits_equal
from oracle import packed_activations as O
from torchft_amd import PackedActivation, PureDistributedDataParallel
from torchft_amd import activations as A

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in DTYPES}
TINY = {t: torch.finfo(t).smallest_normal for t in DTYPES}
ULP32 = 2.0 ** -23


def rounding(v, dtype):
    """Half a step of ``dtype`` at every value (half the least subnormal near zero)."""
    return v.abs() * HALF_STEP[dtype] + TINY[dtype] * HALF_STEP[dtype]


def assert_within(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} vs {tuple(want.shape)}"
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = tuple(int(k) for k in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; at {i} got {got[i]}, "
                             f"want {want[i]} within {tol[i] if torch.is_tensor(tol) else tol}")


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def rows_of(seed, rows, features, dtype):
    x = randn(seed, rows, features) * torch.exp(randn(seed + 1, rows, 1))
    if features > 3:
        x[:, features // 3] *= 40.0
    return x.to(dtype)


def on_gpu(t, device, pad=0, offset=0):
    """t on the GPU, its rows ``pad`` elements apart and its start ``offset`` elements behind an
    allocation's."""
    if t is None:
        return None
    if not pad and not offset:
        return t.to(device)
    rows, n = t.shape
    flat = torch.full((offset + rows * (n + pad) + 8,), 5.0, dtype=t.dtype, device=device)
    view = flat[offset:offset + rows * (n + pad)].view(rows, n + pad)[:, :n]
    view.copy_(t)
    return view


def packed_on_gpu(codes, exponents, features, device, column_scale=None, padding=0):
    values = torch.full((codes.shape[0], (features + 15) // 16 * 16), padding, dtype=torch.uint8)
    values[:, :features] = codes
    return PackedActivation(values.to(device), exponents.to(device), features, column_scale)


def codes_of(p):
    return p.values.view(torch.uint8).cpu()[:, : p.features], p.exponents.cpu()


def assert_same_codes(p, codes, exponents):
    got, got_e = codes_of(p)
    assert torch.equal(got_e, exponents)
    nan = (codes & 0x7F) == 0x7F
    assert torch.equal((got & 0x7F) == 0x7F, nan)
    assert torch.equal(got[~nan], codes[~nan])
    padding = p.values.view(torch.uint8).cpu()[:, p.features:]
    assert not padding.any()


# --- pack and unpack ----------------------------------------------------------------------------

SIZES = [(1, 1), (3, 7), (2, 15), (1, 16), (5, 17), (2, 127), (3, 128), (1, 129), (17, 255), (9, 1000),
         (4, 1153), (64, 256), (33, 2048)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", SIZES)
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
def test_pack_is_bit_exact(device, dtype, rows, features, pad, offset):
    x = rows_of(7 * rows + features, rows, features, dtype)
    codes, exponents = O.pack(x)
    p = A.pack(on_gpu(x, device, pad, offset))
    assert_same_codes(p, codes, exponents)
    want = O.unpack(codes, exponents)
    for out in DTYPES:
        # exact in bf16 and fp32; fp16 rounds once, and holds at most 65504
        assert_bits_equal(p.unpack(out), want.clamp(-65504, 65504).to(out) if out == torch.float16 else want.to(out))
    assert p.unpack().dtype == dtype


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_at_the_ends_of_the_range(device, dtype):
    """Every power of two of the type as a block's largest, next to 1.75 of it; zeros; subnormals."""
    info = torch.finfo(dtype)
    tops = []
    e = int(math.log2(info.smallest_normal)) - 3
    while 2.0 ** e < info.max:
        tops += [2.0 ** e, 1.75 * 2.0 ** e, 1.76 * 2.0 ** e, 1.99 * 2.0 ** e]
        e += 1
    x = torch.zeros(len(tops) + 1, 128, dtype=torch.float64)
    fill = randn(1, len(tops), 128).double()
    x[:-1] = fill / fill.abs().amax(dim=1, keepdim=True)
    x[:-1] *= torch.tensor(tops, dtype=torch.float64)[:, None]
    x = x.clamp(-info.max, info.max).to(dtype)
    codes, exponents = O.pack(x)
    assert_same_codes(A.pack(x.to(device)), codes, exponents)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pack_keeps_nan_and_spares_the_block(device, dtype):
    x = randn(3, 6, 300).to(dtype)
    x[0, 5], x[1, 130], x[2, 299], x[3, 128] = math.nan, math.inf, -math.inf, math.nan
    x[4, :] = math.inf
    codes, exponents = O.pack(x)
    p = A.pack(x.to(device))
    assert_same_codes(p, codes, exponents)
    back = p.unpack().cpu()
    assert torch.equal(torch.isnan(back), ~torch.isfinite(x))
    assert torch.isfinite(back).sum() == torch.isfinite(x).sum()


def test_pack_shapes(device):
    x = randn(1, 2, 3, 4, 130).to(device)
    p = A.pack(x)
    assert p.shape == (2, 3, 4, 130) and p.rows == 24 and p.unpack().shape == x.shape
    one = A.pack(x[0, 0, 0])  # a vector is one row
    assert one.rows == 1 and torch.equal(one.unpack(), p.unpack()[0, 0, 0])
    assert torch.equal(A.pack(x[1, :, 1]).unpack(), p.unpack()[1, :, 1])  # rows with a common stride
    with pytest.raises(ValueError, match="one matrix of rows"):
        A.pack(x[:, 1])
    same = A.pack(x[0, 0, :1].expand(5, 130))  # one row that stands for five
    assert torch.equal(same.unpack(), p.unpack()[0, 0, :1].expand(5, 130))
    for shape in ((0, 130), (5, 0), (0,), (2, 0, 7)):
        e = A.pack(torch.zeros(shape, device=device))
        assert e.unpack().shape == shape


@pytest.mark.parametrize("scale_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_unpack_with_a_column_scale(device, dtype, scale_dtype):
    x = randn(5, 9, 259)
    w = randn(6, 259).to(scale_dtype)
    codes, exponents = O.pack(x)
    p = packed_on_gpu(codes, exponents, 259, device, w.to(device))
    want = O.unpack(codes, exponents) * w.double()
    # one rounding of the product in fp32, one to the output's type
    tol = want.abs() * 2.0 ** -24 + rounding(want, dtype) * (1 + 2.0 ** -20)
    assert_within(p.unpack(dtype), want, tol, "unpack")


# --- norm ---------------------------------------------------------------------------------------

NORM_SIZES = [(1, 1), (2, 3), (5, 64), (3, 129), (4, 512), (7, 513), (6, 1000), (3, 1024), (2, 1025), (5, 2048),
              (3, 2050), (2, 4096), (3, 5001), (2, 8192), (1, 8193), (2, 16384)]


def check_norm(device, rows, features, dtype, weight_dtype, with_residual, pad, offset, seed):
    x = rows_of(seed, rows, features, dtype)
    r = rows_of(seed + 50, rows, features, dtype) if with_residual else None
    w = None if weight_dtype is None else (1 + 0.3 * randn(seed + 2, features)).to(weight_dtype)
    eps = 1e-5
    y, h, p, rstd = A.rms_norm_forward(on_gpu(x, device, pad, offset), None if w is None else w.to(device), eps,
                                       residual=on_gpu(r, device, pad + 2, offset))
    want_y, want_h, n, want_rstd = O.rms_norm(x, w, eps, r)
    if with_residual:  # a single rounding of an exact sum (fp32 adds of fp32 numbers round correctly)
        assert_bits_equal(h, want_h, "h")
    # the sum of squares: at most 32 squares in sequence per lane, then 6 joins in the wavefront
    # and 7 between wavefronts: 45 roundings of 2^-24, halved by the root; mean, root, quotient,
    # product with weight and row: 5 more
    near = (45 / 2 + 5) * 2.0 ** -24
    assert_within(rstd, want_rstd, want_rstd * near, "rstd")
    tol = want_y.abs() * near + rounding(want_y, dtype) * (1 + 2.0 ** -10)
    assert_within(y, want_y, tol, "y")
    kept = O.unpack(*codes_of(p))
    scale = torch.exp2(codes_of(p)[1].double() - 127).repeat_interleave(128, dim=1)[:, :features]
    # half a step of E4M3, of a value that is off by `near`
    tol = torch.maximum(n.abs() * 2.0 ** -4, scale * 2.0 ** -10) * (1 + 2.0 ** -10) + n.abs() * near
    assert_within(kept, n, tol, "packed")
    _, exponents = O.pack(n.float())
    off = (codes_of(p)[1].int() - exponents.int()).abs()
    assert off.max() <= 1 and (off != 0).float().mean() <= 0.02  # only next to 448 * 2^k
    assert not p.values.view(torch.uint8).cpu()[:, features:].any()
    again = A.rms_norm_forward(x.to(device), None if w is None else w.to(device), eps,
                               residual=on_gpu(r, device), pack=False)
    assert again[2] is None
    assert_bits_equal(again[0], y, "y without packing")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", NORM_SIZES)
def test_norm(device, dtype, rows, features):
    check_norm(device, rows, features, dtype, dtype, True, 0, 0, seed=features)


@pytest.mark.parametrize("dtype,weight_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                                (torch.float32, None), (torch.bfloat16, None)])
@pytest.mark.parametrize("rows,features", [(9, 257), (3, 1999)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_forms(device, dtype, weight_dtype, rows, features, with_residual):
    check_norm(device, rows, features, dtype, weight_dtype, with_residual, 3, 1, seed=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1.0, 0.02, 0.001])
def test_norm_without_eps_is_torchs(device, dtype, size):
    """Rows so small that eps decides their norm (at 0.001 it is 12 % of the mean square): the
    module before and after its conversion, both against the definition with fp32's epsilon."""
    x = randn(1, 5, 4096, dtype=dtype, scale=size)
    norm = nn.RMSNorm(4096).to(device, dtype)
    before = norm(x.to(device)).detach()
    after = A.pack_activations(norm)(x.to(device)).detach()
    want = O.rms_norm(x, None, torch.finfo(torch.float32).eps)[0]
    tol = want.abs() * (45 / 2 + 5) * 2.0 ** -24 + rounding(want, dtype) * (1 + 2.0 ** -10)
    assert_within(before, want, tol, "torch's norm")
    assert_within(after, want, tol, "the converted norm")
    assert_bits_equal(A.rms_norm_forward(x.to(device))[0], after)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight_dtype", DTYPES)
def test_norm_module_takes_weights_of_every_type(device, dtype, weight_dtype):
    norm = nn.RMSNorm(130, eps=1e-5).to(device, weight_dtype)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.3 * randn(2, 130))
    x = randn(1, 6, 130, dtype=dtype)
    want = O.rms_norm(x, norm.weight.detach().cpu(), 1e-5)[0]
    tol = want.abs() * (45 / 2 + 5) * 2.0 ** -24 + rounding(want, dtype) * (1 + 2.0 ** -10)
    before = norm(x.to(device))
    after = A.pack_activations(norm)(x.to(device))
    assert before.dtype == after.dtype == dtype
    assert_within(after, want, tol, "y")
    with torch.no_grad():
        assert_bits_equal(norm(x.to(device)), after)
    g = randn(3, 6, 130, dtype=dtype)
    gw, = torch.autograd.grad(after, (norm.weight,), g.to(device))
    packed = getattr(after, A._CARRIED).packed
    n = O.unpack(*codes_of(packed))
    _, want = O.rms_norm_backward(g, n, torch.ones(6), None)
    # six products added in fp32, rounded to fp32 and then to the weight's type
    tol = (g.double() * n).abs().sum(dim=0) * 8 * 2.0 ** -24 + rounding(want, weight_dtype) * (1 + 2.0 ** -10)
    assert gw.dtype == weight_dtype
    assert_within(gw, want, tol, "grad_weight")


def test_norm_of_rows_of_zeros_and_nan(device):
    x = randn(1, 4, 200)
    x[1] = 0.0
    x[2, 7] = math.nan
    x[3, 9] = math.inf
    y, _, p, rstd = A.rms_norm_forward(x.to(device), None, 1e-5)
    y, back = y.cpu(), p.unpack().cpu()
    assert not y[1].any() and not back[1].any() and abs(float(rstd[1]) - 1e-5 ** -0.5) < 1e-3
    assert torch.isnan(y[2]).all() and torch.isnan(back[2]).all()
    assert torch.isnan(y[3, 9]) and not y[3, :9].any()  # inf / inf, the rest over infinity
    assert torch.isfinite(y[0]).all() and torch.isfinite(back[0]).all()
    y, _, p, _ = A.rms_norm_forward(torch.zeros(1, 130, device=device), None, 0.0)
    assert torch.isnan(y).all()  # 0 / 0, as the formula says
    assert not p.values.view(torch.uint8).cpu()[:, 130:].any()


def check_norm_backward(device, rows, features, dtype, weight_dtype, with_h, pad, offset, seed, padding=0):
    gy = (rows_of(seed, rows, features, torch.float32) * 0.05).to(dtype)
    gh = (rows_of(seed + 9, rows, features, torch.float32) * 0.05).to(dtype) if with_h else None
    if rows > 2:
        gy[1] = 0
    w = None if weight_dtype is None else (1 + 0.3 * randn(seed + 2, features)).to(weight_dtype)
    _, _, n, rstd = O.rms_norm(rows_of(seed + 4, rows, features, torch.float32), None, 1e-5)
    if rows * features > 40000:  # the checker's pack is slow; its codes are tested above
        p0 = A.pack(n.float().to(device))
        codes, exponents = codes_of(p0)
    else:
        codes, exponents = O.pack(n.float())
    p = packed_on_gpu(codes, exponents, features, device, None if w is None else w.to(device), padding)
    n = O.unpack(codes, exponents)
    gx, gw = A.rms_norm_backward(on_gpu(gy, device, pad, offset), p, rstd.float().to(device),
                                 grad_h=on_gpu(gh, device, pad, offset))
    want_x, want_w = O.rms_norm_backward(gy, n, rstd.float(), w, gh)
    g = gy.double() if w is None else gy.double() * w.double()
    r = rstd.float().double()[:, None]
    # dot: g rounds once, the products are fused, 45 additions as in the forward pass, one
    # division; grad_x: three more roundings of its terms
    dot_tol = (g * n).abs().sum(dim=1, keepdim=True) / features * 48 * 2.0 ** -24
    terms = g.abs() + n.abs() * (g * n).mean(dim=1, keepdim=True).abs()
    tol = r * (n.abs() * dot_tol + terms * 4 * 2.0 ** -24)
    if with_h:
        tol = tol + gh.double().abs() * 2.0 ** -24
    assert_within(gx, want_x, tol + rounding(want_x, dtype) * (1 + 2.0 ** -10), "grad_x")
    if w is None:
        assert gw is None
        return
    # every row's product is added once, then at most 512 partial sums
    tol = (gy.double() * n).abs().sum(dim=0) * (rows + 20) * 2.0 ** -24
    assert gw.dtype == weight_dtype
    assert_within(gw, want_w, tol + rounding(want_w, weight_dtype) * (1 + 2.0 ** -10), "grad_weight")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", NORM_SIZES + [(2100, 65), (1500, 700), (700, 1030)])
def test_norm_backward(device, dtype, rows, features):
    check_norm_backward(device, rows, features, dtype, dtype, True, 0, 0, seed=features)


@pytest.mark.parametrize("dtype,weight_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32),
                                                (torch.float32, None), (torch.bfloat16, None)])
@pytest.mark.parametrize("rows,features", [(9, 257), (3, 1999)])
@pytest.mark.parametrize("with_h", [False, True])
def test_norm_backward_forms(device, dtype, weight_dtype, rows, features, with_h):
    # the padding of the packed values holds NaN: nothing of it may count
    check_norm_backward(device, rows, features, dtype, weight_dtype, with_h, 3, 1, seed=rows, padding=0x7F)


def test_norm_of_nothing(device):
    w = torch.ones(20, device=device)
    y, _, p, rstd = A.rms_norm_forward(torch.zeros(0, 20, device=device), w)
    assert y.shape == (0, 20) and rstd.shape == (0,)
    gx, gw = A.rms_norm_backward(torch.zeros(0, 20, device=device), p, rstd)
    assert gx.shape == (0, 20) and torch.equal(gw.cpu(), torch.zeros(20))


def test_norm_of_rows_without_features(device):
    """Nothing that a call returns is left as the allocator found it."""
    used = torch.full((1 << 16,), 7.0, device=device)
    del used
    y, h, p, rstd = A.rms_norm_forward(torch.zeros(5, 0, device=device), torch.zeros(0, device=device))
    assert y.shape == h.shape == p.unpack().shape == (5, 0)
    assert torch.isnan(rstd).all()  # 0 / 0
    gx, gw = A.rms_norm_backward(y, p, rstd)
    assert gx.shape == (5, 0) and gw.shape == (0,)


# --- weight gradient ----------------------------------------------------------------------------

PARTS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}


def check_wgrad(device, rows, out_features, features, dtype, out_dtype, scale_dtype, pad, offset, seed, padding=0):
    d = (randn(seed, rows, out_features) * 0.1 * torch.exp(randn(seed + 1, rows, 1))).to(dtype)
    if rows > 3:
        d[2] = 0
    x = rows_of(seed + 3, rows, features, torch.float32)
    codes, exponents = codes_of(A.pack(x.to(device)))
    w = None if scale_dtype is None else (1 + 0.3 * randn(seed + 2, features)).to(scale_dtype)
    p = packed_on_gpu(codes, exponents, features, device, None if w is None else w.to(device), padding)
    n = O.unpack(codes, exponents)
    got = A.linear_weight_grad(on_gpu(d, device, pad, offset), p, dtype=out_dtype)
    want = O.linear_weight_grad(d, n, w)
    # products are exact; every addition may cut a whole step of fp32 (the matrix cores align
    # before they add); rows rounded up to steps of 64 and the joins of the splits
    steps = PARTS[dtype] * (rows + 64) + 64
    tol = O.linear_weight_grad(d.abs(), n.abs(), None if w is None else w.abs()) * steps * ULP32
    assert got.dtype == out_dtype and got.is_contiguous()
    assert_within(got, want, tol + rounding(want, out_dtype) * (1 + 2.0 ** -10), "weight gradient")


WGRAD_SIZES = [(1, 1, 1), (1, 8, 16), (2, 7, 130), (63, 64, 64), (64, 128, 128), (65, 136, 144), (100, 257, 300),
               (130, 1001, 77), (777, 40, 513), (1000, 9, 2000), (2049, 130, 128), (512, 320, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out_features,features", WGRAD_SIZES)
def test_weight_gradient(device, dtype, rows, out_features, features):
    check_wgrad(device, rows, out_features, features, dtype, dtype, None, 0, 0, seed=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("scale_dtype", [None, *DTYPES])
def test_weight_gradient_types(device, dtype, out_dtype, scale_dtype):
    check_wgrad(device, 200, 72, 259, dtype, out_dtype, scale_dtype, 0, 0, seed=5, padding=0x7F)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,offset", [(8, 0), (8, 8), (3, 0), (0, 1), (5, 3)])
@pytest.mark.parametrize("out_features", [64, 61])
def test_weight_gradient_layouts(device, dtype, pad, offset, out_features):
    check_wgrad(device, 150, out_features, 200, dtype, dtype, dtype, pad, offset, seed=8)


def big_wgrad(device, rows, out_features, features, dtype):
    """Against a product in fp64 on the GPU."""
    g = torch.Generator(device=device).manual_seed(rows)
    d = (torch.randn(rows, out_features, generator=g, device=device) * 0.01).to(dtype)
    p = A.pack(torch.randn(rows, features, generator=g, device=device))
    n = p.unpack(torch.float32).double()
    want = torch.mm(d.double().t().contiguous(), n)
    bound = torch.mm(d.double().abs().t().contiguous(), n.abs())
    tol = bound * (PARTS[dtype] * (rows + 64) + 64) * ULP32 + rounding(want, dtype) * (1 + 2.0 ** -10)
    got = A.linear_weight_grad(d, p).double()
    assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("rows,out_features,features,dtype", [
    (300, 4096, 2560, torch.bfloat16), (1000, 2300, 4100, torch.bfloat16), (200, 3000, 4000, torch.float16),
    (200, 2824, 3001, torch.float32), (4096, 1024, 4096, torch.bfloat16), (70, 14336, 4096, torch.bfloat16)])
def test_weight_gradient_of_large_layers(device, rows, out_features, features, dtype):
    big_wgrad(device, rows, out_features, features, dtype)


def plan_of(device, rows, out_features, features, dtype):
    """Pieces' workspace of a weight gradient whose rows are read as they lie."""
    d = torch.empty(16, device=device, dtype=dtype)
    return A._native.lib().tft_linear_weight_grad_workspace(d.data_ptr(), rows, out_features, features, out_features,
                                                          (features + 15) // 16 * 16, A._DTYPES[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out_features,features,cut", [
    (1, 64, 64, False), (65, 136, 144, None), (70, 14336, 4096, None), (300, 4096, 2560, None),
    (1000, 1000, 768, True), (4096, 1024, 4096, True), (2049, 130, 128, None), (40, 61, 77, False)])
def test_weight_gradient_keeps_every_bit(device, dtype, rows, out_features, features, cut):
    """One row of gradients of full significands against powers of two: every output is a product,
    and exact.  Large and small tiles, whole and cut ones; the row lies in each part of a step."""
    if cut is not None and out_features % 8 == 0:
        assert bool(plan_of(device, rows, out_features, features, dtype)) == cut
    g = torch.Generator().manual_seed(rows)
    signs = torch.randint(0, 2, (1, features), generator=g) * 2 - 1
    x_row = torch.exp2(torch.randint(-6, 7, (1, features), generator=g).float()) * signs
    bits = torch.randint(0, 1 << 30, (1, out_features), generator=g).double() * 2.0 ** -30 + 1.0  # 1 .. 2
    small = [] if dtype == torch.float16 else [2.0 ** -104]
    for at, size in [(0, 0.5), (rows - 1, 1.0), (rows // 2, 2.0 ** -8), *((rows // 3, s) for s in small)]:
        d_row = (bits * size).to(dtype)
        d = torch.zeros(rows, out_features, dtype=dtype, device=device)
        x = torch.zeros(rows, features, device=device)
        d[at], x[at] = d_row[0].to(device), x_row[0].to(device)
        got = A.linear_weight_grad(d, A.pack(x), dtype=torch.float32)
        want = d[at].double()[:, None] * x[at].double()  # 24 bits times a power of two
        assert torch.equal(got.double(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 17, 40])
def test_weight_gradient_of_few_rows(device, dtype, rows):
    """Bounds tight enough to tell a missing part of the gradient from a rounding."""
    d = randn(rows, rows, 72).to(dtype)
    p = A.pack(randn(rows + 1, rows, 130).to(device))
    n = O.unpack(*codes_of(p))
    got = A.linear_weight_grad(d.to(device), p, dtype=torch.float32)
    want = O.linear_weight_grad(d, n)
    assert_within(got, want, O.weight_grad_bound(d, n, PARTS[dtype]) + want.abs() * 2.0 ** -24, "weight gradient")


@pytest.mark.parametrize("dtype,stride", [(torch.bfloat16, 1 << 24), (torch.float16, 1 << 24), (torch.float32, 1 << 23),
                                          (torch.bfloat16, (1 << 24) - 8), (torch.float32, (1 << 23) + 1)])
def test_weight_gradient_of_rows_far_apart(device, dtype, stride):
    """A step's slice of a gradient that holds many steps: 32 MB and more from row to row."""
    d = randn(2, 70, 64, dtype=dtype).to(device)
    p = A.pack(randn(1, 70, 200).to(device))
    far = torch.empty(69 * stride + 64, dtype=dtype, device=device).as_strided((70, 64), (stride, 1))
    far.copy_(d)
    assert_bits_equal(A.linear_weight_grad(far, p), A.linear_weight_grad(d, p))
    steps = far.unsqueeze(1)  # [70, 1, 64]: the rows are a view's
    assert_bits_equal(A.linear_weight_grad(steps, p), A.linear_weight_grad(d, p))


def test_weight_gradient_of_expanded_and_empty(device):
    p = A.pack(randn(1, 90, 200).to(device))
    row = randn(2, 1, 64, dtype=torch.bfloat16).to(device)
    assert torch.equal(A.linear_weight_grad(row.expand(90, 64), p),
                       A.linear_weight_grad(row.expand(90, 64).contiguous(), p))
    none = A.pack(torch.zeros(0, 200, device=device))
    assert torch.equal(A.linear_weight_grad(torch.zeros(0, 8, device=device), none).cpu(), torch.zeros(8, 200))
    assert A.linear_weight_grad(torch.zeros(90, 0, device=device), p).shape == (0, 200)
    assert A.linear_weight_grad(torch.zeros(3, 8, device=device), A.pack(torch.zeros(3, 0, device=device))).shape == (8, 0)


def test_weight_gradient_with_infinities(device):
    """An infinity of the gradient reaches its own output row alone, as NaN where it meets zero."""
    for dtype in DTYPES:
        d = randn(1, 70, 16).to(dtype)
        d[5, 3] = math.inf
        d[6, 9] = math.nan
        x = randn(2, 70, 130)
        x[5, 7] = 0.0
        p = A.pack(x.to(device))
        got = A.linear_weight_grad(d.to(device), p, dtype=torch.float32).cpu()
        n5 = p.unpack().cpu()[5]
        want = torch.where(n5 == 0, torch.tensor(math.nan), torch.copysign(torch.tensor(math.inf), n5))
        assert torch.equal(torch.isnan(got[3]), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got[3][ok], want[ok])
        assert torch.isnan(got[9]).all()
        rest = [i for i in range(16) if i not in (3, 9)]
        assert torch.isfinite(got[rest]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 7), (200, 130), (5000, 33), (17, 5000), (4097, 1000)])
def test_column_sum(device, dtype, rows, columns):
    x = randn(rows, rows, columns).to(dtype)
    want = x.double().sum(dim=0)
    tol = x.double().abs().sum(dim=0) * (rows + 40) * 2.0 ** -24 + rounding(want, dtype) * (1 + 2.0 ** -10)
    assert_within(A.column_sum(on_gpu(x, device, 3, 1)), want, tol, "column sum")
    assert torch.equal(A.column_sum(torch.zeros(0, columns, device=device)).cpu(), torch.zeros(columns))


# --- long buffers, streams, graphs ----------------------------------------------------------------


def test_offsets_past_32_bits(device):
    """4.4e9 elements: the last rows are packed, read back and multiplied from where they lie."""
    rows, features, tail = (1 << 21) + 5, 2096, 70
    x = torch.zeros(rows, features, dtype=torch.bfloat16, device=device)
    x[-tail:] = randn(1, tail, features, dtype=torch.bfloat16).to(device)
    x[0] = 3.0
    p = A.pack(x)
    small = A.pack(x[-tail:].clone())
    assert torch.equal(p.values[-tail:].view(torch.uint8), small.values.view(torch.uint8))
    assert torch.equal(p.exponents[-tail:], small.exponents)
    back = p.unpack()
    assert torch.equal(back[-tail:], small.unpack()) and bool((back[0] == 3.0).all())
    assert not bool(back[1:-tail].any())
    d = x[:, :8].contiguous()
    d[0] = 0
    big = A.linear_weight_grad(d, p, dtype=torch.float32)
    want = O.linear_weight_grad(d[-tail:].cpu(), small.unpack().cpu())
    tol = O.linear_weight_grad(d[-tail:].cpu().abs(), small.unpack().cpu().abs()) * 400 * ULP32
    assert_within(big, want, tol, "weight gradient")  # the other rows are zeros and add exactly
    del back, big
    wide = A.linear_weight_grad(x, _tail_packed(p, 16), dtype=torch.float32)  # long gradients, few features
    sixteen = small.unpack().cpu()[:, :16]
    full = x[-tail:].cpu()
    want = O.linear_weight_grad(full, sixteen) + 3.0 * 3.0
    tol = (O.linear_weight_grad(full.abs(), sixteen.abs()) + 9.0) * 400 * ULP32
    assert_within(wide, want, tol, "weight gradient of long rows")


def _tail_packed(p, features):
    return PackedActivation(p.values[:, :features].contiguous(), p.exponents[:, :1].contiguous(), features)


def test_output_past_32_bits(device):
    """2.4e9 elements of a weight gradient: its last rows against the checker."""
    rows, out_features, features = 20, 590_000, 4096
    d = torch.zeros(rows, out_features, dtype=torch.bfloat16, device=device)
    d[:, -70:] = randn(1, rows, 70, dtype=torch.bfloat16).to(device)
    p = A.pack(randn(2, rows, features).to(device))
    got = A.linear_weight_grad(d, p)
    n = p.unpack().cpu()
    want = O.linear_weight_grad(d[:, -70:].cpu(), n)
    tol = O.linear_weight_grad(d[:, -70:].cpu().abs(), n.abs()) * 200 * ULP32
    assert_within(got[-70:], want, tol + rounding(want, torch.bfloat16) * (1 + 2.0 ** -10), "last rows")
    assert not bool(got[:-70].any())


def test_norm_offsets_past_32_bits(device):
    rows, features = (1 << 20) + 3, 4160
    x = torch.ones(rows, features, dtype=torch.bfloat16, device=device)
    x[-3:] = randn(1, 3, features, dtype=torch.bfloat16).to(device)
    y, _, p, rstd = A.rms_norm_forward(x, None, 1e-5)
    sy, _, sp, srstd = A.rms_norm_forward(x[-3:].clone(), None, 1e-5)
    assert torch.equal(y[-3:], sy) and torch.equal(rstd[-3:], srstd)
    assert torch.equal(p.values[-3:].view(torch.uint8), sp.values.view(torch.uint8))
    gx, _ = A.rms_norm_backward(x, p, rstd)
    sgx, _ = A.rms_norm_backward(x[-3:].clone(), sp, srstd)
    assert torch.equal(gx[-3:], sgx)


def test_norm_of_more_rows_than_a_launch_holds(device):
    """2^26 rows of a wavefront each are 2^32 threads, one more than a dispatch can have."""
    rows, features, tail = (1 << 26) + 5, 8, 70
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(rows, features, generator=g, device=device, dtype=torch.bfloat16)
    r = torch.randn(rows, features, generator=g, device=device, dtype=torch.bfloat16)
    w = (1 + 0.3 * randn(2, features)).to(device)
    y, h, p, rstd = A.rms_norm_forward(x, w, 1e-5, r)
    for part in (slice(rows - tail, rows), slice((1 << 26) - 40, (1 << 26) - 4), slice(0, tail)):
        sy, sh, sp, srstd = A.rms_norm_forward(x[part].contiguous(), w, 1e-5, r[part].contiguous())
        assert_bits_equal(y[part], sy)
        assert_bits_equal(h[part], sh)
        assert_bits_equal(rstd[part], srstd)
        assert_bits_equal(p.values[part].view(torch.uint8), sp.values.view(torch.uint8))
        assert_bits_equal(p.exponents[part], sp.exponents)
    gx, gw = A.rms_norm_backward(x, p, rstd, r)
    sgx, _ = A.rms_norm_backward(x[-tail:].contiguous(), A.rms_norm_forward(x[-tail:], w, 1e-5, r[-tail:])[2],
                                 rstd[-tail:].contiguous(), r[-tail:])
    assert_bits_equal(gx[-tail:], sgx)


def test_norm_of_more_wide_rows_than_a_launch_holds(device):
    """2^25 rows of two wavefronts each; the rows of x overlap, each starts one element on."""
    rows, features, tail = (1 << 25) + 3, 520, 70
    g = torch.Generator(device=device).manual_seed(1)
    x = torch.randn(rows + features, generator=g, device=device, dtype=torch.bfloat16).as_strided((rows, features), (1, 1))
    y, _, _, rstd = A.rms_norm_forward(x, None, 1e-5, pack=False)
    for part in (slice(rows - tail, rows), slice((1 << 25) - 40, (1 << 25)), slice(0, tail)):
        sy, _, _, srstd = A.rms_norm_forward(x[part].contiguous(), None, 1e-5, pack=False)
        assert_bits_equal(y[part], sy)
        assert_bits_equal(rstd[part], srstd)
    del x, y
    torch.cuda.empty_cache()


def test_packing_of_more_blocks_than_a_launch_holds(device):
    """2^30 blocks of sixteen lanes; unpacking reaches the same at half as many.  One small whole
    number a block: it is kept exactly."""
    rows = (1 << 30) + 70
    x = torch.randint(1, 8, (rows, 1), device=device, dtype=torch.int8).bfloat16()
    p = A.pack(x)
    back = p.unpack()
    assert torch.equal(back, x)
    small = A.pack(x[-50:])
    assert torch.equal(p.values[-50:].view(torch.uint8), small.values.view(torch.uint8))
    del x, p, back
    torch.cuda.empty_cache()


def test_column_sum_of_more_columns_than_a_launch_holds(device):
    columns = (1 << 27) + 40
    x = torch.randint(-7, 8, (10, columns), device=device, dtype=torch.int8).bfloat16()
    assert torch.equal(A.column_sum(x, torch.float32), x.float().sum(dim=0))
    torch.cuda.empty_cache()


def test_calls_run_on_the_current_stream_and_repeat(device):
    x, d = randn(1, 300, 1000).to(device), randn(2, 300, 257).to(device)
    w = torch.ones(1000, device=device)

    def all_of_it():
        y, _, p, rstd = A.rms_norm_forward(x, w, 1e-5)
        gx, gw = A.rms_norm_backward(x, p, rstd)
        return y, p.unpack(), gx, gw, A.linear_weight_grad(d, p), A.column_sum(d)

    want = all_of_it()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [all_of_it() for _ in range(3)]
    other = all_of_it()  # at the same time on the first stream
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for g in (*got, other):
        for a, b in zip(g, want):
            assert_bits_equal(a, b)  # no sum depends on the order in which work ends


def small_block(dtype, device):
    torch.manual_seed(0)
    return nn.Sequential(nn.RMSNorm(192, eps=1e-5), nn.Linear(192, 320), nn.SiLU(), nn.Linear(320, 192),
                         nn.RMSNorm(192, eps=1e-5), nn.Linear(192, 100, bias=False)).to(device, dtype)


def test_a_captured_layer_packs_what_its_replays_read(device):
    """The graph holds the layer and not the norm: new rows are written into the norm's output."""
    norm, lin = A.RMSNorm(130).to(device), A.Linear(130, 8).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lin(norm(randn(1, 6, 130).to(device)))
    torch.cuda.current_stream().wait_stream(side)
    y = norm(randn(1, 6, 130).to(device))
    assert A._native.lib().tft_capture_id(torch.cuda.current_stream().cuda_stream) == 0
    kept, ids = [], []
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            out = lin(y)
            z = norm(y)
            again = lin(z)  # the graph's own norm packs for this one
            ids.append(A._native.lib().tft_capture_id(torch.cuda.current_stream().cuda_stream))
            kept.append((out.grad_fn.saved_tensors[1], again.grad_fn.saved_tensors[1]))
            assert kept[-1][1].data_ptr() == getattr(z, A._CARRIED).packed.values.data_ptr()
            del out, z, again
    assert 0 not in ids and ids[0] != ids[1] and A._UNKNOWN_CAPTURE not in ids
    for k in range(3):
        with torch.no_grad():
            y.copy_(randn(k + 7, 6, 130))
        for graph, (values, normed) in zip(graphs, kept):
            graph.replay()
            torch.cuda.synchronize()
            assert_bits_equal(values.view(torch.uint8), A.pack(y.detach()).values.view(torch.uint8))
            assert_bits_equal(normed.view(torch.uint8),
                              A.rms_norm_forward(y.detach(), norm.weight)[2].values.view(torch.uint8))


def test_captured_steps_replay(device):
    model = A.pack_activations(small_block(torch.bfloat16, device))
    x = torch.zeros(130, 192, dtype=torch.bfloat16, device=device)
    target = torch.zeros(130, 100, dtype=torch.bfloat16, device=device)
    params = list(model.parameters())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad((model(x) * target).sum(), params)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs, grads = [], [], []
    for _ in range(2):  # two graphs of the same step, each with workspaces of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = model(x)
            gr = torch.autograd.grad((out * target).sum(), params)
        graphs.append(g)
        outs.append(out.detach())
        del out  # no autograd graph of these leaves outlives its capture
        grads.append(gr)
    for k in range(4):
        x.copy_(randn(k, 130, 192, dtype=torch.bfloat16))
        target.copy_(randn(k + 9, 130, 100, dtype=torch.bfloat16))
        graphs[k % 2].replay()
        if k >= 2:
            graphs[(k + 1) % 2].replay()
        torch.cuda.synchronize()
        want = model(x)
        want_grads = torch.autograd.grad((want * target).sum(), params)
        for which in ([k % 2] if k < 2 else [0, 1]):
            assert_bits_equal(outs[which], want)
            for a, b in zip(grads[which], want_grads):
                assert_bits_equal(a, b)


def test_graphed_callables(device):
    """torch's own capture of a module, forward and backward apart."""
    model = A.pack_activations(small_block(torch.bfloat16, device))
    again = A.pack_activations(small_block(torch.bfloat16, device))
    sample = torch.zeros(130, 192, dtype=torch.bfloat16, device=device, requires_grad=True)
    graphed = torch.cuda.make_graphed_callables(model, (sample,))
    for k in range(4):
        x = randn(k, 130, 192, dtype=torch.bfloat16).to(device).requires_grad_()
        g = randn(k + 9, 130, 100, dtype=torch.bfloat16).to(device)
        out = graphed(x)
        got = [t.clone() for t in torch.autograd.grad(out, [x, *model.parameters()], g)]
        out = out.detach().clone()
        torch.cuda.synchronize()
        plain = again(x)
        want = torch.autograd.grad(plain, [x, *again.parameters()], g)
        assert_bits_equal(out, plain)
        for a, b in zip(got, want):
            assert_bits_equal(a, b)


def test_captured_layers_on_two_streams(device):
    """A capture that forks: the layer reads the norm's rows on the other stream, in every replay."""
    norm, lin = A.RMSNorm(256).to(device), A.Linear(256, 16).to(device)
    x = torch.zeros(40, 256, device=device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lin(norm(x))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = norm(x)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = lin(y)
        torch.cuda.current_stream().wait_stream(side)
        values, result = out.grad_fn.saved_tensors[1], out.detach()
        assert values.data_ptr() == getattr(y, A._CARRIED).packed.values.data_ptr()
        del y, out
    for k in range(3):
        x.copy_(randn(k, 40, 256))
        graph.replay()
        torch.cuda.synchronize()
        plain = norm(x)
        assert_bits_equal(result, lin(plain))
        assert_bits_equal(values.view(torch.uint8), getattr(plain, A._CARRIED).packed.values.view(torch.uint8))


# --- autograd, modules and the wrappers -----------------------------------------------------------


def test_norm_gradients_reach_both_inputs(device):
    x = randn(1, 2, 5, 130).to(device).requires_grad_()
    r = randn(2, 2, 5, 130).to(device).requires_grad_()
    w = (1 + 0.1 * randn(3, 130)).to(device).requires_grad_()
    gy, gh = randn(4, 2, 5, 130).to(device), randn(5, 2, 5, 130).to(device)
    y, h, p = A.rms_norm(x, w, 1e-5, r)
    assert p.shape == (2, 5, 130) and not p.values.requires_grad
    gx, gr, gw = torch.autograd.grad((y * gy).sum() + (h * gh).sum(), (x, r, w))
    n = O.unpack(*codes_of(p))
    rstd = 1.0 / (h.detach().double().cpu().reshape(10, 130).pow(2).mean(dim=1) + 1e-5).sqrt()
    want, want_w = O.rms_norm_backward(gy.cpu().reshape(10, 130), n, rstd, w.detach().cpu(), gh.cpu().reshape(10, 130))
    assert torch.equal(gx, gr)
    assert_within(gx.reshape(10, 130), want, want.abs() * 1e-5 + 1e-5, "grad_x")
    assert_within(gw, want_w, want_w.abs() * 1e-5 + 1e-5, "grad_weight")
    # against the norm without packing: the kept rows are off by 2^-4 of themselves, and by their
    # part of the row the mean is taken over
    ref = torch.nn.functional.rms_norm(x + r, (130,), w, 1e-5)
    fx, = torch.autograd.grad((ref * gy).sum() + ((x + r) * gh).sum(), (x,))
    assert float((gx - fx).norm() / fx.norm()) < 2.0 ** -4
    y2, h2, p2 = A.rms_norm(x, w, 1e-5, r)  # only h is read: y's gradient is absent
    gx2, = torch.autograd.grad((h2 * gh).sum(), (x,))
    assert torch.equal(gx2, gh)
    with torch.no_grad():
        y3, h3, p3 = A.rms_norm(x, w, 1e-5, r)
        assert p3 is None and torch.equal(y3, y2) and torch.equal(h3, h2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(5, 130), (2, 3, 130), (130,)])
def test_linear_keeps_the_forward_pass(device, dtype, shape):
    x = randn(1, *shape).to(device, dtype).requires_grad_()
    w = (randn(2, 40, 130) * 0.1).to(device, dtype).requires_grad_()
    b = randn(3, 40).to(device, dtype).requires_grad_()
    out = A.linear(x, w, b)
    plain = nn.functional.linear(x, w, b)
    assert_bits_equal(out, plain)
    g = randn(4, *out.shape).to(device, dtype)
    gx, gw, gb = torch.autograd.grad(out, (x, w, b), g)
    fx, = torch.autograd.grad(plain, (x,), g)
    assert gx.shape == x.shape
    assert_within(gx, fx.cpu(), fx.cpu().double().abs() * HALF_STEP[dtype] * 4 + 1e-6, "grad_x")
    rows = g.reshape(-1, 40)
    p = A.pack(x.detach().reshape(-1, 130))
    assert_bits_equal(gw, A.linear_weight_grad(rows, p))
    assert_bits_equal(gb, A.column_sum(rows))


def test_linear_inputs_of_any_layout(device):
    w = randn(2, 7, 40).to(device).requires_grad_()
    base = randn(1, 40, 6, 5).to(device)
    for x in (base.permute(1, 2, 0), base.permute(2, 1, 0), base[:, 0].t(), base[:, 0, 0].expand(3, 40)):
        out = A.linear(x, w)
        gw, = torch.autograd.grad(out.sum(), (w,))  # an expanded gradient
        want, = torch.autograd.grad(A.linear(x.contiguous(), w).sum(), (w,))
        assert_bits_equal(gw, want)
    frozen = w.detach()
    x = randn(4, 3, 40).to(device).requires_grad_()
    out = A.linear(x, frozen)
    assert torch.autograd.grad(out.sum(), (x,))[0].shape == x.shape
    assert not A.linear(x.detach(), frozen).requires_grad


def test_packed_norm_output_is_shared_by_the_layers_behind_it(device):
    norm, a, b = (A.pack_activations(m.to(device)) for m in (nn.RMSNorm(130), nn.Linear(130, 8), nn.Linear(130, 9)))
    x = randn(1, 6, 130).to(device)
    y = norm(x)
    packed = getattr(y, A._CARRIED)[0]
    before = torch.cuda.memory_allocated()
    za, zb = a(y), b(y)
    kept = torch.cuda.memory_allocated() - before
    assert kept <= 2 * 512  # the two outputs, and no further packed rows
    ga, gb = randn(2, 6, 8).to(device), randn(3, 6, 9).to(device)
    gwa, gwb = torch.autograd.grad((za * ga).sum() + (zb * gb).sum(), (a.weight, b.weight))
    assert_bits_equal(gwa, A.linear_weight_grad(ga, packed))
    assert_bits_equal(gwb, A.linear_weight_grad(gb, packed))
    with torch.no_grad():
        y.mul_(2.0)  # written to since: the layer packs what it sees
    gw, = torch.autograd.grad((a(y) * ga).sum(), (a.weight,))
    assert_bits_equal(gw, A.linear_weight_grad(ga, A.pack(y.detach())))


@pytest.mark.parametrize("autocast", [False, True])
def test_layers_that_read_one_activation_keep_one_copy(device, autocast):
    """Query, key and value projections behind a norm that is not ours, as one after another and as
    a whole: the bytes that they keep, their gradients, and what is left once they are gone."""
    rows, features = 64, 1024
    ln = nn.LayerNorm(features).to(device)
    layers = [A.Linear(features, 16).to(device) for _ in range(3)]
    y = ln(randn(1, rows, features).to(device))
    grads = [randn(k, rows, 16).to(device) for k in range(3)]
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
        [layer(y) for layer in layers]  # whatever the products allocate once
        before = torch.cuda.memory_allocated()
        outs = [layer(y) for layer in layers]
        kept = {o.grad_fn.saved_tensors[1].data_ptr() for o in outs}
        nothing = [nn.functional.linear(y.detach(), layer.weight.detach()) for layer in layers]
        assert len(kept) == 1
    if not autocast:  # the outputs, and their values and exponents
        assert torch.cuda.memory_allocated() - before <= 6 * rows * 16 * 4 + rows * (features + features // 128)
    del nothing
    got = torch.autograd.grad([(o * g).sum() for o, g in zip(outs, grads)], [layer.weight for layer in layers])
    cast = y.detach().bfloat16() if autocast else y.detach()
    for gw, g in zip(got, grads):
        assert_bits_equal(gw, A.linear_weight_grad(g.to(cast.dtype), A.pack(cast)).float())
    del outs, got, gw
    weak = getattr(y, A._SHARED)
    assert weak.values() is None and weak.exponents() is None
    with torch.no_grad():
        y.mul_(2.0)
    first = layers[0](y)
    with torch.no_grad():
        y.mul_(2.0)  # the first layer's rows are no longer y's
    second = layers[1](y)
    gw, = torch.autograd.grad((second * grads[1]).sum(), (layers[1].weight,))
    assert_bits_equal(gw, A.linear_weight_grad(grads[1], A.pack(y.detach())))
    gw, = torch.autograd.grad((first * grads[0]).sum(), (layers[0].weight,))
    assert_bits_equal(gw, A.linear_weight_grad(grads[0], A.pack(y.detach() / 2)))


def test_layers_on_other_streams_pack_for_themselves(device):
    """Nothing makes the second stream wait for what the first one packed."""
    layers = [A.Linear(256, 16).to(device) for _ in range(2)]
    y = torch.relu(randn(1, 40, 256).to(device).requires_grad_())
    first = layers[0](y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = layers[1](y)
    a, b = first.grad_fn.saved_tensors[1], second.grad_fn.saved_tensors[1]
    torch.cuda.synchronize()
    assert a.data_ptr() != b.data_ptr()
    assert_bits_equal(a.view(torch.uint8), b.view(torch.uint8))


def test_views_of_a_norms_output_share_its_rows(device):
    norm, layer = A.RMSNorm(256).to(device), A.Linear(256, 16).to(device)
    y = norm(randn(1, 2, 20, 256).to(device))
    kept = getattr(y, A._CARRIED).packed.values
    g = randn(2, 40, 16).to(device)
    for whole in (y.view(-1, 256), y.flatten(0, 1), y.unsqueeze(0), y.view(4, 10, 256)):
        out = layer(whole)
        assert out.grad_fn.saved_tensors[1].data_ptr() == kept.data_ptr()
        gw, = torch.autograd.grad((out.view(40, 16) * g).sum(), (layer.weight,))
        assert_bits_equal(gw, A.linear_weight_grad(g, getattr(y, A._CARRIED).packed))
    square = A.RMSNorm(16).to(device)(randn(1, 16, 16).to(device))
    narrow = A.Linear(16, 8).to(device)
    for part in (square[:15], square[1:], square.t(), square.view(16, 1, 16).expand(16, 2, 16), square.view(256, 1),
                 square.view(8, 32)):  # other rows, another order, rows twice, other rows' ends
        lin = narrow if part.shape[-1] == 16 else A.Linear(part.shape[-1], 8).to(device)
        out = lin(part)
        g = randn(3, *out.shape).to(device)
        gw, = torch.autograd.grad((out * g).sum(), (lin.weight,))
        rows = part.detach().reshape(-1, part.shape[-1]).contiguous()
        assert_bits_equal(gw, A.linear_weight_grad(g.reshape(-1, 8), A.pack(rows)))
    flat = y.view(-1, 256)
    with torch.no_grad():
        flat.mul_(2.0)  # a write to one is a write to all
    for t in (flat, y.view(-1, 256)):
        gw, = torch.autograd.grad((layer(t) * randn(2, 40, 16).to(device)).sum(), (layer.weight,))
        assert_bits_equal(gw, A.linear_weight_grad(randn(2, 40, 16).to(device), A.pack(t.detach())))


def test_a_shared_activation_saves_and_loads_as_a_tensor(device):
    y = torch.relu(randn(1, 40, 256).to(device).requires_grad_())
    layer = A.Linear(256, 16).to(device)
    out = layer(y)
    file = io.BytesIO()
    torch.save(y, file)
    file.seek(0)
    again = torch.load(file, weights_only=True)
    assert torch.equal(again, y)
    assert_bits_equal(layer(torch.relu(again)), out)
    assert_bits_equal(layer(again), out)


def test_a_norms_output_saves_and_loads_as_a_tensor(device):
    """Its packed rows are not written with it: safe loading would refuse their class."""
    norm, layer = A.RMSNorm(256).to(device), A.Linear(256, 16).to(device)
    y = norm(randn(1, 40, 256).to(device))
    file = io.BytesIO()
    torch.save(y, file)
    assert len(file.getvalue()) < 40 * 256 * 4 + 4096
    file.seek(0)
    again = torch.load(file, weights_only=True)
    assert torch.equal(again, y)
    assert_bits_equal(layer(again), layer(y))


def test_packed_rows_saved_on_the_host_and_modules_with_hooks(device):
    x, g = randn(1, 33, 192).to(device), randn(2, 33, 100).to(device)
    model = A.pack_activations(small_block(torch.float32, device))
    want = torch.autograd.grad(model(x), list(model.parameters()), g)
    with torch.autograd.graph.save_on_cpu():
        out = model(x)
    got = torch.autograd.grad(out, list(model.parameters()), g)
    for m in model:
        m.register_full_backward_hook(lambda *a: None)  # its inputs and outputs are views then
        m.register_forward_hook(lambda *a: None)
    inp = x.clone().requires_grad_()
    hooked = torch.autograd.grad(model(inp), list(model.parameters()), g)
    for a, b, c in zip(got, hooked, want):
        assert_bits_equal(a, c)
        assert_bits_equal(b, c)


def test_input_buffers_are_packed_by_every_layer(device):
    """A program's own buffer may be rewritten in ways that torch does not count."""
    layers = [A.Linear(256, 16).to(device) for _ in range(2)]
    x = randn(1, 40, 256).to(device)
    first = layers[0](x)
    x.data.copy_(randn(2, 40, 256))
    g = randn(3, 40, 16).to(device)
    gw, = torch.autograd.grad((layers[1](x) * g).sum(), (layers[1].weight,))
    assert_bits_equal(gw, A.linear_weight_grad(g, A.pack(x)))
    del first


def test_modules_without_gradients_and_without_rows(device):
    model = A.pack_activations(small_block(torch.float32, device))
    x = randn(1, 5, 192).to(device)
    want = model(x).detach()
    with torch.inference_mode():
        assert torch.equal(model(x), want)
    with torch.no_grad():
        assert torch.equal(model(x), want)
    empty = torch.zeros(0, 192, device=device, requires_grad=True)
    grads = torch.autograd.grad(model(empty).sum(), [empty, *model.parameters()])
    assert grads[0].shape == (0, 192) and not any(bool(g.any()) for g in grads)
    norm = A.pack_activations(nn.RMSNorm(192, elementwise_affine=False).to(device))
    row = x[0].clone().requires_grad_()  # one row, no weight
    y = norm(row)
    assert y.shape == (192,) and torch.autograd.grad(y.sum(), row)[0].shape == (192,)


def test_two_threads_at_once(device):
    """Calls keep nothing between them: two threads on two streams get what one gets."""
    import threading

    data = [(randn(k, 400, 640).to(device), randn(k + 9, 400, 136, dtype=torch.float16).to(device)) for k in (1, 2)]

    def work(x, d):
        y, _, p, rstd = A.rms_norm_forward(x, None, 1e-5)
        return y, A.rms_norm_backward(x, p, rstd)[0], A.linear_weight_grad(d, p), p.unpack()

    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[k] = work(*data[k])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # shown by the assertion below
            errors.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert_bits_equal(a, b)


def test_writing_to_a_norms_weight_before_the_backward_pass_is_an_error(device):
    norm, lin = A.RMSNorm(64).to(device), A.Linear(64, 8).to(device)
    out = lin(norm(randn(1, 4, 64).to(device)))
    with torch.no_grad():
        norm.weight.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_writing_to_a_norms_weight_before_the_layer_behind_it(device):
    """The packed rows are to be multiplied with the weight that the norm's output was made with."""
    norm, lin = A.RMSNorm(130).to(device), A.Linear(130, 8).to(device)
    g = randn(2, 6, 8).to(device)
    y = norm(randn(1, 6, 130).to(device))
    with torch.no_grad():
        norm.weight.mul_(3.0)
    gw, = torch.autograd.grad((lin(y) * g).sum(), (lin.weight,))
    assert_bits_equal(gw, A.linear_weight_grad(g, A.pack(y.detach())))
    out = A.rms_norm(randn(1, 6, 130).to(device), norm.weight)
    A.linear(out.y, lin.weight, packed=out.packed)
    with torch.no_grad():
        norm.weight.mul_(2.0)
    with pytest.raises(ValueError, match="written to since"):
        A.linear(out.y, lin.weight, packed=out.packed)


def test_giving_a_norms_output_other_storage(device):
    norm, lin = A.RMSNorm(130).to(device), A.Linear(130, 8).to(device)
    y, g = norm(randn(1, 6, 130).to(device)), randn(2, 6, 8).to(device)
    kept = y.detach()
    y.data = randn(5, 6, 130).to(device)  # torch does not count this as a write
    gw, = torch.autograd.grad((lin(y) * g).sum(), (lin.weight,))
    assert_bits_equal(gw, A.linear_weight_grad(g, A.pack(y.detach())))
    assert not torch.equal(kept, y)
    for made in (A.RMSNorm(64).to(device), torch.relu):  # the same address, turned around
        y = made(randn(1, 64, 64).to(device).requires_grad_())
        first = A.Linear(64, 8).to(device)
        out = first(y)
        y.data = y.data.t()
        g = randn(2, 64, 8).to(device)
        gw, = torch.autograd.grad((first(y) * g).sum(), (first.weight,))
        assert_bits_equal(gw, A.linear_weight_grad(g, A.pack(y.detach().contiguous())))
        del out


def test_packed_rows_outlive_the_stream_that_reads_them(device):
    """A layer on another stream than its norm's: after y.record_stream, as torch asks, the packed
    rows behind y are not handed out again while that stream may still read them."""
    norm, lin = A.RMSNorm(4096).to(device), A.Linear(4096, 8).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        lin(norm(torch.ones(64, 4096, device=device)))
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    y = norm(torch.ones(8192, 4096, device=device))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        out = lin(y)
    y.record_stream(side)
    packed = getattr(y, A._CARRIED).packed
    kept = packed.values.data_ptr()
    assert out.grad_fn.saved_tensors[1].data_ptr() == kept
    del y, out, packed
    fresh = [torch.empty(8192, 4096, dtype=torch.uint8, device=device) for _ in range(3)]
    assert not side.query()  # it is still asleep
    assert kept not in [t.data_ptr() for t in fresh]
    torch.cuda.synchronize()


def test_autocast(device):
    lin = A.Linear(130, 16).to(device)
    x = randn(1, 9, 130).to(device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = lin(x)
        plain = nn.functional.linear(x, lin.weight, lin.bias)
    assert out.dtype == torch.bfloat16
    assert_bits_equal(out, plain)
    out.float().sum().backward()
    assert lin.weight.grad.dtype == torch.float32 and lin.bias.grad.dtype == torch.float32
    want = A.linear_weight_grad(torch.ones(9, 16, dtype=torch.bfloat16, device=device), A.pack(x.bfloat16()))
    assert torch.equal(lin.weight.grad, want.float())


def test_autocast_leaves_64_bits_alone(device):
    x = randn(1, 3, 8).to(device)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert nn.functional.linear(x.double(), x.double()).dtype == torch.float64
        with pytest.raises(TypeError, match="float64"):
            A.Linear(8, 4).to(device).double()(x.double())
        with pytest.raises(TypeError, match="float64"):
            A.linear(x.double(), randn(2, 4, 8).to(device))


class Averaging:
    """A manager whose all-reduce halves the gradient, as two participants with one idle would."""

    def __init__(self):
        self.calls = 0

    def allreduce(self, t):
        self.calls += 1
        t.div_(2.0)
        f = torch.futures.Future()
        f.set_result(t)
        return f


class Block(nn.Module):
    """A pre-norm residual block: the second norm takes the sum."""

    def __init__(self, width):
        super().__init__()
        self.first, self.second = nn.RMSNorm(width, eps=1e-5), nn.RMSNorm(width, eps=1e-5)
        self.a, self.b = nn.Linear(width, 2 * width), nn.Linear(2 * width, width)
        self.head = nn.Linear(width, 50, bias=False)

    def forward(self, x):
        y = self.b(torch.nn.functional.silu(self.a(self.first(x))))
        if type(self.second) is A.RMSNorm:
            z, _ = self.second(y, x)
        else:
            z = self.second(y + x)
        return self.head(z)


@pytest.mark.parametrize("dtype,near", [(torch.float32, 2.0 ** -4), (torch.bfloat16, 2.0 ** -4 + 2.0 ** -6)])
@pytest.mark.parametrize("wrapper", ["ddp", "pure"])
def test_wrapped_model_trains_on_packed_activations(device, dtype, near, wrapper):
    """The model's outputs stay what they are (the norm's rounding apart) and every parameter's
    gradient is within E4M3's half step of the one from full activations: each is a sum of products
    with kept values, of which every one is off by at most 2^-4 of itself, in norm."""
    from torchft_amd import DistributedDataParallel

    torch.manual_seed(3)
    plain = Block(256).to(device, dtype)
    import copy
    model = copy.deepcopy(plain)
    x, target = randn(1, 4, 33, 256, dtype=dtype).to(device), randn(2, 4, 33, 50, dtype=dtype).to(device)
    want = plain(x)
    (want * target).sum().backward()
    manager = Averaging()
    if wrapper == "ddp":
        wrapped = DistributedDataParallel(manager, model, packed_activations=True)
    else:
        wrapped = PureDistributedDataParallel(manager, model, packed_activations=True)
    assert type(model.a) is A.Linear and type(model.first) is A.RMSNorm
    out = wrapped(x)
    assert float(((out - want).norm() / want.norm()).detach()) < 8 * HALF_STEP[dtype]
    (out * target).sum().backward()
    assert manager.calls >= 1
    for (name, p), q in zip(model.named_parameters(), plain.parameters()):
        off = float((2 * p.grad - q.grad).norm() / q.grad.norm())
        assert off < near, f"{name}: {off}"


@pytest.mark.parametrize("reentrant", [False, True])
@pytest.mark.parametrize("autocast", [False, True])
def test_checkpointed_layers(device, reentrant, autocast):
    """The second forward pass packs what the first one did: the gradients are the same bits."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(1)
    before, block = nn.LayerNorm(192).to(device), A.pack_activations(small_block(torch.float32, device))
    q, k = A.Linear(192, 100).to(device), A.Linear(192, 100).to(device)
    params = [before.weight, *block.parameters(), q.weight, k.weight]

    def part(x):  # an input that several layers read, and one behind a norm
        return block(x) + q(x) * k(x)

    def step(run):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            out = run(before(randn(2, 33, 192).to(device)))
        return out.detach(), torch.autograd.grad((out.float() * randn(3, 33, 100).to(device)).sum(), params)

    out, want = step(part)
    if reentrant:
        for p in params:
            p.grad = None
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            again = checkpoint(part, before(randn(2, 33, 192).to(device)), use_reentrant=True)
        (again.float() * randn(3, 33, 100).to(device)).sum().backward()
        got = [p.grad for p in params]
    else:
        again, got = step(lambda x: checkpoint(part, x, use_reentrant=False))
    assert_bits_equal(again, out)
    for a, b in zip(got, want):
        assert_bits_equal(a, b)


@pytest.mark.parametrize("outer_step", [False, True])
def test_converted_model_under_localsgd_and_diloco(device, outer_step):
    """Two replicas, a sync behind every step: the parameters that the kernels write, the norm's
    weights among them, are those that the next step's gradients are made with."""
    import copy

    from oracle import replica_sync as sync
    from test_gpu_api import cpu, peer_world
    from torch import optim
    from torchft_amd import DiLoCo, LocalSGD, Manager, ProcessGroupLocalReplicas, StaticQuorum

    torch.manual_seed(2)
    plain = nn.Sequential(nn.RMSNorm(192), nn.Linear(192, 64), nn.SiLU(), nn.Linear(64, 10)).to(device)
    model = A.pack_activations(copy.deepcopy(plain))
    peers, lookup = peer_world(model, 2)
    g = torch.Generator().manual_seed(7)
    for q in peers[0].parameters():
        q.data.add_((torch.randn(q.shape, generator=g) * 1e-2).to(device))
    pg = ProcessGroupLocalReplicas(rank=0, world_size=2, peer_lookup=lookup)
    manager = Manager(pg=pg, load_state_dict=None, state_dict=None, min_replica_size=2, use_async_quorum=False,
                      quorum_client=StaticQuorum(0, 2))
    inner = optim.SGD(model.parameters(), lr=0.1)
    if outer_step:
        wrapped = DiLoCo(manager, model, inner, optim.SGD(model.parameters(), lr=0.7, momentum=0.9, nesterov=True),
                         sync_every=1)
    else:
        wrapped = LocalSGD(manager, model, inner, sync_every=1)
    seen = {}
    with wrapped:
        perform = wrapped._perform_sync

        def recording():
            seen["local"] = cpu(p.data for p in model.parameters())
            perform()

        wrapped._perform_sync = recording
        backup, bufs = cpu(wrapped._backup_parameters.values()), None
        for step in range(3):
            fresh = copy.deepcopy(model)
            x, t = randn(step, 40, 192).to(device), randn(step + 9, 40, 10).to(device)
            inner.zero_grad()
            (model(x) * t).sum().backward()
            (fresh(x) * t).sum().backward()
            for p, q in zip(model.parameters(), fresh.parameters()):
                assert_bits_equal(p.grad, q.grad)
            inner.step()  # the sync runs behind it
            replicas = [seen["local"], cpu(q.data for q in peers[0].parameters())]
            if outer_step:
                want = sync.diloco_perform_sync(replicas, backup, bufs, [True] * 2, 2, True, lr=0.7, momentum=0.9,
                                                nesterov=True)
                bufs = want["momentum"]
            else:
                want = sync.localsgd_perform_sync(replicas, backup, [True, True], 2, True)
            backup = want["backup"] if outer_step else want["params"]
            for p, w in zip(model.parameters(), want["params"]):
                assert_bits_equal(p.data, w)
    assert manager.current_step() == 3
    manager.shutdown(wait=False)
