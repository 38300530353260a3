"""Packed activations without a GPU: the checker against definitions and differences, the
refusals of the Python functions and of the C entries, and the module conversion."""

import copy
import ctypes
import math
import pickle
import subprocess
import sys

import pytest
import torch
from torch import nn

from conftest import REPO_ROOT
from oracle import packed_activations as O
from torchft_amd import PackedActivation, PureDistributedDataParallel, _native, pack_activations
from torchft_amd import activations as A


# --- the checker ------------------------------------------------------------------------------


def test_e4m3_numbers_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).float().double()
    got = O.e4m3_values()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok])


def test_rounding_to_e4m3_is_torchs():
    g = torch.Generator().manual_seed(1)
    grid = O.e4m3_values()[:127]
    ties = (grid[1:] + grid[:-1]) / 2
    v = torch.cat([torch.randn(5000, generator=g).double() * 30, grid, ties, -ties,
                   torch.rand(3000, generator=g).double() * 2.0 ** -6])
    v = v.float().double().clamp(-448, 448)
    want = v.float().to(torch.float8_e4m3fn).float().double()
    assert torch.equal(O.e4m3_values()[O.to_e4m3(v).long()], want)


@pytest.mark.parametrize("top,exponent", [
    (448.0, 127), (448.0 * (1 + 2 ** -20), 128), (1.75, 119), (1.7500001, 120), (1.0, 119),
    (0.0, 10), (2.0 ** -127, 10), (3.4e38, 246), (math.inf, 10), (math.nan, 10),
])
def test_block_exponent(top, exponent):
    x = torch.zeros(1, 5, dtype=torch.float32)
    x[0, 3] = top
    codes, e = O.pack(x)
    assert e.tolist() == [[exponent]]
    if not math.isfinite(top):
        assert codes[0, 3] & 0x7F == 0x7F


def test_packed_values_are_exact_in_bf16():
    grid = O.e4m3_values()
    grid = grid[~torch.isnan(grid)]
    for e in (10, 11, 64, 127, 200, 246):
        v = grid * 2.0 ** (e - 127)
        assert torch.equal(v.float().to(torch.bfloat16).double(), v)
        nonzero = v[v != 0].abs()
        assert float(nonzero.min()) >= 2.0 ** -126  # a normal number


def test_checkers_gradients_are_differences():
    g = torch.Generator().manual_seed(3)
    x, r, gy, gh = (torch.randn(3, 10, generator=g, dtype=torch.float64) for _ in range(4))
    w = torch.randn(10, generator=g, dtype=torch.float64)

    def loss(x, r, w):
        y, h, _, _ = O.rms_norm(x, w, 1e-3, r)
        return float((y * gy).sum() + (h * gh).sum())

    _, _, n, rstd = O.rms_norm(x, w, 1e-3, r)
    gx, gw = O.rms_norm_backward(gy, n, rstd, w, gh)
    step = 1e-6
    for i in range(3):
        for j in range(10):
            d = torch.zeros_like(x)
            d[i, j] = step
            # central differences: step^2 of the third derivative, 2^-53 / step of rounding
            assert abs((loss(x + d, r, w) - loss(x - d, r, w)) / (2 * step) - float(gx[i, j])) < 1e-7
            assert abs((loss(x, r + d, w) - loss(x, r - d, w)) / (2 * step) - float(gx[i, j])) < 1e-7
    for j in range(10):
        d = torch.zeros_like(w)
        d[j] = step
        assert abs((loss(x, r, w + d) - loss(x, r, w - d)) / (2 * step) - float(gw[j])) < 1e-7


@pytest.mark.parametrize("dtype,parts", [(torch.float32, 3), (torch.float16, 2)])
@pytest.mark.parametrize("rows", [1, 3, 8])
def test_bound_of_the_weight_gradient_tells_a_missing_part(dtype, parts, rows):
    """A gradient cut into one bf16 part too few is outside of the bound that the GPU's is held to."""
    g = torch.Generator().manual_seed(rows)
    d = torch.randn(rows, 40, generator=g).to(dtype)
    x = O.unpack(*O.pack(torch.randn(rows, 30, generator=g)))
    want, bound = O.linear_weight_grad(d, x), O.weight_grad_bound(d, x, parts)
    assert torch.equal(O.bf16_parts(d, parts), d.double())
    short = O.linear_weight_grad(O.bf16_parts(d, parts - 1), x)
    assert ((short - want).abs() > bound).double().mean() > 0.5
    assert ((d.float().t() @ x.float()).double() - want).abs().le(bound).all()


# --- refusals -----------------------------------------------------------------------------------


def test_no_cpu_path():
    x = torch.zeros(4, 128)
    for call in (lambda: A.pack(x), lambda: A.rms_norm(x), lambda: A.rms_norm_forward(x),
                 lambda: A.column_sum(x), lambda: A.linear(x, torch.zeros(3, 128)),
                 lambda: PackedActivation(x, x, 128), lambda: A.Linear(128, 3)(x),
                 lambda: A.RMSNorm(128)(x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(TypeError, match="expected a tensor"):
        A.pack([1.0])


def test_layer_names_what_is_no_tensor():
    for x in (None, [1.0], 3):
        with pytest.raises(TypeError, match="linear: x: expected a tensor"):
            A.Linear(128, 3)(x)


class FakeGpu(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks run, nothing is launched."""

    is_cuda = True


def gpu(t):
    return t.as_subclass(FakeGpu)


def test_pack_refuses():
    with pytest.raises(TypeError, match="float32, bfloat16 and float16"):
        A.pack(gpu(torch.zeros(2, 3, dtype=torch.float64)))
    with pytest.raises(ValueError, match="consecutive"):
        A.pack(gpu(torch.zeros(4, 8).t()))
    with pytest.raises(ValueError, match="one matrix of rows"):
        A.pack(gpu(torch.zeros(4, 6, 8).transpose(0, 1)))
    with pytest.raises(ValueError, match="scalar"):
        A.pack(gpu(torch.tensor(1.0)))


def test_packed_form_is_checked():
    v, e = torch.zeros(2, 144, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    with pytest.raises(TypeError, match="float8"):
        PackedActivation(gpu(v.float()), gpu(e), 130)
    with pytest.raises(ValueError, match="144"):
        PackedActivation(gpu(v[:, :128].contiguous()), gpu(e), 130)
    with pytest.raises(ValueError, match="contiguous"):
        PackedActivation(gpu(torch.zeros(2, 160, dtype=torch.uint8)[:, :144]), gpu(e), 130)
    with pytest.raises(ValueError, match="exponents"):
        PackedActivation(gpu(v), gpu(e[:, :1].contiguous()), 130)
    with pytest.raises(ValueError, match="130 consecutive"):
        PackedActivation(gpu(v), gpu(e), 130, column_scale=gpu(torch.zeros(129)))
    with pytest.raises(ValueError, match="does not hold"):
        PackedActivation(gpu(v), gpu(e), 130, shape=(3, 130))
    with pytest.raises(TypeError, match="float64"):
        PackedActivation(gpu(v), gpu(e), 130, dtype=torch.float64)
    p = PackedActivation(gpu(v), gpu(e), 130)
    assert (p.rows, p.shape, p.dtype, p.nbytes) == (2, (2, 130), torch.bfloat16, 2 * 146)


def test_packed_form_is_copied_and_pickled():
    """A copy's scale counts its writes from nought; one that was void stays void."""
    def form():
        scale = torch.zeros(130).add_(1.0)
        return A._trusted(torch.ones(2, 144, dtype=torch.uint8), torch.ones(2, 2, dtype=torch.uint8), 130, scale,
                          (1, 2, 130), torch.float16)

    for copied in (copy.copy, copy.deepcopy, lambda p: pickle.loads(pickle.dumps(p))):
        p = form()
        q = copied(p)
        assert q._scale_is_as_packed() and (q.shape, q.dtype, q.features) == (p.shape, p.dtype, p.features)
        assert torch.equal(q.values, p.values) and torch.equal(q.exponents, p.exponents)
        q.column_scale.mul_(2.0)
        assert not q._scale_is_as_packed()
        p = form()
        p.column_scale.mul_(2.0)
        assert not copied(p)._scale_is_as_packed()
        p.column_scale = None
        p._scale_version = None
        assert copied(p)._scale_is_as_packed() and copied(p).column_scale is None


def test_norm_refuses():
    x = gpu(torch.zeros(2, 16, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="16 consecutive"):
        A.rms_norm_forward(x, gpu(torch.zeros(15)))
    with pytest.raises(TypeError, match="expected torch.bfloat16 or float32"):
        A.rms_norm_forward(x, gpu(torch.zeros(16, dtype=torch.float16)))
    with pytest.raises(ValueError, match="eps"):
        A.rms_norm_forward(x, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        A.rms_norm_forward(x, eps=math.nan)
    with pytest.raises(ValueError, match="residual"):
        A.rms_norm_forward(x, residual=gpu(torch.zeros(2, 16)))
    with pytest.raises(ValueError, match="at most 16384"):
        A.rms_norm_forward(gpu(torch.zeros(1, 16385)))


def packed_of(rows, features, scale=None):
    return PackedActivation(gpu(torch.zeros(rows, (features + 15) // 16 * 16, dtype=torch.uint8)),
                            gpu(torch.zeros(rows, -(-features // 128), dtype=torch.uint8)), features, scale)


def test_backward_functions_refuse():
    p = packed_of(3, 16, gpu(torch.zeros(16)))
    rstd = gpu(torch.zeros(3))
    with pytest.raises(ValueError, match="rows"):
        A.rms_norm_backward(gpu(torch.zeros(2, 16)), p, rstd)
    with pytest.raises(ValueError, match="rstd"):
        A.rms_norm_backward(gpu(torch.zeros(3, 16)), p, gpu(torch.zeros(2)))
    with pytest.raises(ValueError, match="grad_h"):
        A.rms_norm_backward(gpu(torch.zeros(3, 16)), p, rstd, grad_h=gpu(torch.zeros(3, 17)))
    with pytest.raises(ValueError, match="packed 3"):
        A.linear_weight_grad(gpu(torch.zeros(4, 8)), p)
    with pytest.raises(TypeError, match="float64"):
        A.linear_weight_grad(gpu(torch.zeros(3, 8)), p, dtype=torch.float64)
    with pytest.raises(ValueError, match="does not fit"):
        A.linear(gpu(torch.zeros(3, 15)), gpu(torch.zeros(4, 16)))
    with pytest.raises(ValueError, match="packed is of shape"):
        A.linear(gpu(torch.zeros(4, 16)), gpu(torch.zeros(4, 16)), packed=p)


def test_c_entries_refuse_without_a_gpu():
    lib = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    err = lib.tft_last_error
    ok = dict(values=at, exponents=at, x=at, rows=1, features=130, stride=130, pitch=144, dtype=0)

    def pack(**kw):
        return lib.tft_pack_e4m3(*{**ok, **kw}.values(), None)

    assert pack(dtype=_native.TFT_F64) == -2 and b"not fp32, bf16 or fp16" in err()
    assert pack(rows=-1) == -1 and b"negative size" in err()
    assert pack(stride=-1) == -1 and b"row stride" in err()
    assert pack(pitch=128) == -1 and b"pitch" in err()
    assert pack(pitch=145) == -1 and b"pitch" in err()
    assert pack(pitch=272) == -1 and b"pitch" in err()
    assert pack(features=100, pitch=144) == -1 and b"last block" in err()
    assert pack(values=at + 8) == -1 and b"16 bytes" in err()
    assert pack(x=at + 2) == -1 and b"misaligned" in err()
    assert pack(x=None) == -1 and pack(values=None) == -1 and pack(exponents=None) == -1
    assert pack(rows=1 << 31) == -2 and b"2^31" in err()
    assert pack(rows=1 << 30, features=512, pitch=512) == -2 and b"blocks" in err()
    assert pack(rows=0, values=None, x=None) == 0 and pack(features=0, pitch=0) == 0

    assert lib.tft_unpack_e4m3(None, at, at, None, 1, 130, 144, 0, 0, None) == -1
    assert lib.tft_unpack_e4m3(at, at, at, at + 1, 1, 130, 144, 1, 0, None) == -1
    assert lib.tft_unpack_e4m3(at, at, at, at, 1, 130, 144, 3, 0, None) == -2
    assert lib.tft_unpack_e4m3(None, None, None, None, 0, 130, 144, 0, 0, None) == 0

    def norm(y=at, h=None, x=at, residual=None, weight=at, features=130, eps=1e-5, wt=0, t=0, rows=1):
        return lib.tft_rms_norm(y, h, at, at, at, x, residual, weight, rows, features, features, 0,
                                (features + 15) // 16 * 16, eps, wt, t, None)

    assert norm(features=16385) == -2 and b"at most 16384" in err()
    assert norm(eps=-1.0) == -1 and norm(eps=math.nan) == -1
    assert norm(residual=at) == -1 and b"come together" in err()
    assert norm(h=at) == -1 and norm(y=None) == -1 and norm(x=at + 1) == -1
    assert norm(wt=2, t=1) == -2 and b"dtype or fp32" in err()
    assert norm(weight=at + 2) == -1 and norm(rows=0) == 0

    def back(ws=at, ws_bytes=1 << 20, gw=at, gx=at, rstd=at, rows=3, wt=0):
        return lib.tft_rms_norm_backward(gx, gw, ws, ws_bytes, at, None, at, at, rstd, at, rows, 130, 130, 0,
                                         144, wt, 0, None)

    need = lib.tft_rms_norm_backward_workspace(3, 130)
    assert need == 130 * 4  # one workgroup for four rows
    assert back(ws_bytes=need - 1) == -1 and b"workspace" in err()
    assert back(ws=None) == -1 and back(gx=None) == -1 and back(rstd=None) == -1
    assert back(wt=1) == -2

    assert lib.tft_column_sum(None, at, 4096, at, 3, 8, 8, 0, 0, None) == -1
    assert lib.tft_column_sum(at, at, 31, at, 3, 8, 8, 0, 0, None) == -1 and b"32 are needed" in err()

    def wgrad(out=at, ws=at, ws_bytes=1 << 30, g=at, rows=64, o=64, features=130, stride=64, pitch=144,
              ot=1, st=0, t=1, scale=None):
        return lib.tft_linear_weight_grad(out, ws, ws_bytes, g, at, at, scale, rows, o, features, stride, pitch,
                                          ot, st, t, None)

    assert wgrad(t=3) == -2 and wgrad(ot=3) == -2 and wgrad(st=9, scale=at) == -2
    assert wgrad(out=None) == -1 and wgrad(out=at + 8) == -1 and wgrad(g=None) == -1
    assert wgrad(stride=-64) == -1 and wgrad(o=-1) == -1
    assert wgrad(stride=1 << 25, rows=2) == -2 and b"too long" in err()
    assert wgrad(o=63, stride=63, ws_bytes=0) == -1 and b"8192 are needed" in err()
    assert wgrad(o=63, ws=None) == -1 and wgrad(o=63, ws=at + 8) == -1
    assert wgrad(o=0) == 0 and wgrad(features=0, pitch=0) == 0
    space = lib.tft_linear_weight_grad_workspace
    for t in range(3):
        assert space(at, 64, 64, 130, 64, 144, t) == 0  # aligned rows are read as they lie
    assert space(at, 64, 63, 130, 63, 144, 0) == 64 * 64 * 4
    assert space(at + 2, 64, 64, 130, 64, 144, 1) == 64 * 64 * 2
    assert space(at, 64, 63, 130, 63, 144, 1) == 64 * 64 * 2
    assert space(at, 64, 64, 130, 0, 144, 1) == 64 * 64 * 2  # one row that stands for all
    assert space(at, 0, 64, 130, 64, 144, 1) == 0
    # one small tile and 16 tokens: nothing to cut; 4096 tokens: pieces, in fp32
    assert space(at, 16, 128, 128, 128, 128, 1) == 0
    assert space(at, 4096, 128, 128, 128, 128, 1) % (128 * 128 * 4) == 0
    assert space(at, 4096, 128, 128, 128, 128, 1) >= 2 * 128 * 128 * 4


def test_weight_gradients_of_more_tiles_than_a_launch_holds_are_refused():
    """2^27 tiles of 512 threads: over the 2^32 threads of a dispatch (16 TB of gradient)."""
    lib = _native.lib()
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    rc = lib.tft_linear_weight_grad(at, at, 1 << 62, at, at, at, None, 1, 1 << 23, 1 << 20, 1 << 23, 1 << 20,
                                    1, 0, 1, None)
    assert rc == -2 and b"tiles" in lib.tft_last_error()


@pytest.mark.parametrize("rows,out_features,features,dtype,tile,tiles,pieces", [
    (8192, 4096, 4096, 1, 256, 256, 1), (8192, 1024, 4096, 1, 256, 64, 4), (4096, 2048, 2048, 2, 256, 64, 4),
    (16384, 1000, 1000, 0, 256, 16, 16), (4096, 1024, 4096, 1, 128, 256, 2), (1024, 768, 768, 1, 128, 36, 4),
    (1000, 1008, 768, 0, 128, 48, 5)])
def test_how_weight_gradients_are_cut(rows, out_features, features, dtype, tile, tiles, pieces):
    """The pieces that the figures beside the kernel speak of, by the workspace that they take."""
    got = _native.lib().tft_linear_weight_grad_workspace(4096, rows, out_features, features, out_features,
                                                         (features + 15) // 16 * 16, dtype)
    assert got == (tiles * pieces * tile * tile * 4 if pieces > 1 else 0)


# --- modules ------------------------------------------------------------------------------------


def test_imports_under_a_torch_without_gpu_support():
    """Such a build lacks the names that ask for the current stream and device."""
    code = ("import torch\n"
            "for name in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    delattr(torch._C, name)\n"
            "import torchft_amd\n"
            "torchft_amd.pack_activations(torch.nn.Linear(2, 2))\n")
    done = subprocess.run([sys.executable, "-c", code], cwd=REPO_ROOT, capture_output=True, text=True, timeout=110)
    assert done.returncode == 0, done.stderr


class Odd(nn.Linear):
    pass


def make_model():
    return nn.Sequential(nn.RMSNorm(16), nn.Linear(16, 8), nn.ReLU(), Odd(8, 8), nn.RMSNorm((4, 8)),
                         nn.LayerNorm(8), nn.RMSNorm(20000), nn.MultiheadAttention(8, 2))


def test_conversion_takes_plain_linears_and_norms_only():
    model = make_model()
    state = {k: v.clone() for k, v in model.state_dict().items()}
    assert pack_activations(model) is model
    assert [type(m) for m in model][:7] == [A.RMSNorm, A.Linear, nn.ReLU, Odd, nn.RMSNorm, nn.LayerNorm, nn.RMSNorm]
    assert type(model[7].out_proj) is not A.Linear
    after = model.state_dict()
    assert list(after) == list(state) and all(torch.equal(after[k], state[k]) for k in state)
    pack_activations(model)  # once more changes nothing
    assert type(model[1]) is A.Linear
    assert type(pack_activations(nn.Linear(2, 2))) is A.Linear
    for other in (copy.deepcopy(model), pickle.loads(pickle.dumps(model))):
        assert type(other[0]) is A.RMSNorm and type(other[1]) is A.Linear
        assert torch.equal(other[1].weight, model[1].weight)


def test_pure_ddp_converts_on_request():
    assert type(PureDistributedDataParallel(None, nn.Linear(2, 2)).module) is nn.Linear
    assert type(PureDistributedDataParallel(None, nn.Linear(2, 2), packed_activations=True).module) is A.Linear
