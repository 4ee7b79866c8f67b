"""Long sums of the product and of its gradients: the tensor cores cut an accumulator's last bits off at every addition, which must not add
up to anything that a result in 16 bits shows, nor keep a wait of the kernel beyond its limit."""

import pytest
import torch

from lplb_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
# A result is off by half a step of its type, and by what its sum is off: 6e-9 of it per product that the tensor cores add up, products of
# one sign, so 4.9e-5 for the parts of 8192 that a result in float16 is taken in, 3.9e-4 for 65536 in bfloat16, and 2^-24 at most for each of
# up to 512 parts, 3e-5.  Here 1.8e-4 and 9.8e-4 are allowed.
OFF = {F16: 2.0**-11 * 9 / 8 + 2.0**-13, BF16: 2.0**-8 * 9 / 8 + 2.0**-11}


def _positive(*shape, scale, dtype, seed):
    """Numbers of one sign with all their bits, so that every addition cuts the same way."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (scale * (0.5 + torch.rand(*shape, device="cuda", generator=g))).to(dtype)


def _in_64(a, b):
    """a @ b.T in 64 bits, a stretch of the sum at a time."""
    out = torch.zeros(a.shape[0], b.shape[0], dtype=torch.float64, device="cuda")
    for at in range(0, a.shape[1], 1 << 17):
        out += a[:, at : at + (1 << 17)].double() @ b[:, at : at + (1 << 17)].double().T
    return out


def _check(got, want, dtype):
    off = ((got.double() - want) / want).abs().max().item()
    assert got.dtype == dtype and off <= OFF[dtype] and ops.check() == 0, off


@pytest.mark.parametrize("dtype,length", [(F16, 1 << 20), (F16, 1 << 22), (BF16, 1 << 22)])
@pytest.mark.parametrize("m", [1, 48])
def test_forward_of_few_rows(m, dtype, length):
    a, b = _positive(m, length, scale=1e-2, dtype=dtype, seed=1), _positive(24, length, scale=1e-1, dtype=dtype, seed=2)
    _check(ops.matmul(a, b), _in_64(a, b), dtype)


@pytest.mark.parametrize("dtype,length", [(F16, 1 << 20), (BF16, 1 << 22)])
@pytest.mark.parametrize("activation,n", [(None, 24), ("swiglu", 256)])
def test_forward_of_groups(activation, n, dtype, length):
    a, b = _positive(40, length, scale=1e-2, dtype=dtype, seed=1), _positive(2, n, length, scale=1e-3, dtype=dtype, seed=2)
    rows = torch.tensor([33, 5], dtype=torch.int32, device="cuda")
    got = ops.matmul(a, b, activation=activation, rows=rows)
    want = torch.cat([_in_64(a[:33], b[0]), _in_64(a[33:38], b[1])])
    if activation == "swiglu":  # both factors are of some 10 or more: silu is the factor itself there
        want = torch.nn.functional.silu(want[:, :128]) * want[:, 128:]
        assert ((got[:38].double() - want) / want).abs().max() <= OFF[dtype] + 3 * (OFF[dtype] - 2.0**-11 * (1 if dtype == F16 else 8))
    else:
        _check(got[:38], want, dtype)
    assert not got[38:].any() and ops.check() == 0


@pytest.mark.parametrize("dtype,length", [(F16, 1 << 20), (BF16, 1 << 22)])
@pytest.mark.parametrize("grouped", [False, True])
def test_input_gradient(grouped, dtype, length):
    a = torch.zeros(20, 8, dtype=dtype, device="cuda").requires_grad_()
    b, d = _positive(length, 8, scale=1e-1, dtype=dtype, seed=1), _positive(20, length, scale=1e-2, dtype=dtype, seed=2)
    more = {}
    if grouped:
        more["rows"] = torch.tensor([20], dtype=torch.int32, device="cuda")
    (da,) = torch.autograd.grad(ops.matmul(a, b[None] if grouped else b, **more), a, d)
    _check(da, _in_64(d, b.T), dtype)


def _weight_gradient(groups, dtype, n=8, out_dtype=None):
    m = sum(max(r, 0) for r in groups)
    a, d = _positive(m, 16, scale=1e-1, dtype=dtype, seed=1), _positive(m, n, scale=1e-2, dtype=out_dtype or dtype, seed=2)
    one = len(groups) == 1
    b = torch.zeros(*(() if one else (len(groups),)), n, 16, dtype=dtype, device="cuda").requires_grad_()
    more = {} if one else {"rows": torch.tensor(groups, dtype=torch.int32, device="cuda")}
    (db,) = torch.autograd.grad(ops.matmul(a, b, out_dtype=out_dtype, **more), b, d)
    at = 0
    for e, r in enumerate(groups):
        r = max(r, 0)
        if r == 0:
            assert not db[e].any()
        else:
            _check(db if one else db[e], _in_64(d[at : at + r].T, a[at : at + r].T), dtype)
        at += r
    return a, d, db


@pytest.mark.parametrize("n", [8, 300])
@pytest.mark.parametrize("dtype,length", [(F16, (1 << 20) + 5), (BF16, 1 << 22)])
def test_weight_gradient(n, dtype, length):
    _weight_gradient([length], dtype, n)


@pytest.mark.parametrize("dtype,groups", [(F16, [5, 1 << 20, 0, 16_384, 16_385, -3, 300, 65_537]), (BF16, [1 << 22, 0, 131_072, 131_073, 77])])
def test_weight_gradient_of_groups(dtype, groups):
    """Long ones beside short and empty ones: every matrix is written, once."""
    _weight_gradient(groups, dtype)


@pytest.mark.parametrize("dtype,part", [(F16, 8192), (BF16, 65536)])
def test_lengths_around_a_part(dtype, part):
    """One block more or less than whole parts, long tiles beside short ones and behind one another, on few and many tiles per SM."""
    _weight_gradient([part - 1, part, part + 1, 5, 2 * part, 2 * part + 1, 64, 3 * part - 63], dtype)
    _weight_gradient([2 * part + 65, 100, part + 64, part + 64, 7], dtype, n=1024)
    _weight_gradient([part + 1], dtype, n=1029)


@pytest.mark.parametrize("activation,n,off", [("silu", 264, False), ("silu", 264, True), ("swiglu", 512, False), ("swiglu", 512, True)])
@pytest.mark.parametrize("groups", [None, [700, 0, 1, 299, 300]])
def test_long_sums_with_everything_behind_them(groups, activation, n, off):
    """Bias, activation, residual and what backward needs, results that leave by whole words or not, several long tiles for every pair; against the
    sums of a result in 32 bits, which are taken in parts of 512."""
    m, k = 1300, 3 * 8192 + 200
    g = torch.Generator(device="cuda").manual_seed(n)
    normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    lead = () if groups is None else (len(groups),)
    cols = n // 2 if activation == "swiglu" else n
    residual = normal(m, cols + 1).half()
    args = {
        "a": normal(m, k).half(),
        "b": (normal(*lead, n, k) * k**-0.5).half(),
        "bias": normal(*lead, n),
        "residual": residual[:, 1:] if off else residual[:, 1:].contiguous(),
        "activation": activation,
        "rows": None if groups is None else torch.tensor(groups, dtype=torch.int32, device="cuda"),
    }
    want = ops.matmul(**{**args, "residual": args["residual"].float()}, out_dtype=torch.float32)
    bias = args["bias"].requires_grad_()
    got = ops.matmul(**args)
    # random signs: a sum is off by far less than its half step here, 2^-11 of what is summed at the end
    size = want.abs() + args["residual"].float().abs() + 1
    assert ((got.float() - want).abs() <= size * (2.0**-11 + 2.0**-13)).all()
    d = normal(m, cols)
    (kept,) = torch.autograd.grad(got, bias, d.half())
    whole = ops.matmul(**{**args, "residual": args["residual"].float()}, out_dtype=torch.float32)
    (right,) = torch.autograd.grad(whole, bias, d.half().float())
    # z is off by what its sum is: 7e-6 of its magnitudes' norm and more, and as much the slopes, summed over up to 1300 rows
    assert ((kept - right).norm() / right.norm()).item() <= 2.0**-13
    with torch.no_grad():
        assert torch.equal(ops.matmul(**args), got) and ops.check() == 0


def test_weight_gradient_of_results_in_32_bits():
    _weight_gradient([1 << 20], F16, out_dtype=torch.float32)
    _weight_gradient([100, 1 << 20], F16, out_dtype=torch.float32)


def test_the_same_bits_every_time():
    _, _, first = _weight_gradient([70_000, 300, 200_000], F16)
    for _ in range(3):
        assert torch.equal(_weight_gradient([70_000, 300, 200_000], F16)[2], first)


def test_a_sum_over_a_thousand_million_rows_stays_within_its_waits():
    """One tile sums them all: some 17 million blocks, seconds of work for a wait of two seconds at most."""
    m = 2**30
    a = torch.zeros(m, 8, dtype=BF16, device="cuda")
    a[::4] = 1
    a[-3:] = 2
    a.requires_grad_()
    b = torch.ones(1, 8, dtype=BF16, device="cuda").requires_grad_()
    out = ops.matmul(a, b)
    (db,) = torch.autograd.grad(out, b, torch.ones(1, 1, dtype=BF16, device="cuda").expand(m, 1))
    assert torch.equal(db, torch.full((1, 8), float(m // 4), dtype=BF16, device="cuda")) and ops.check() == 0
