"""The product with an epilogue on the GPU, forward and backward, against its definition in 64 bits with derived bounds."""

import pytest
import torch
from test_ops_matmul import ACTIVATIONS, compare, make_case, refusals, run

from lplb_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(m, n, k, groups=None, activation=None, bias=None, residual=False, dtype=BF16, out_dtype=BF16, seed=0):
    args, dout = make_case(m, n, k, groups, activation, bias, residual, dtype, out_dtype, seed + m + n + k, "cuda")
    got = run(args, dout)
    compare(got, args, dout)
    # without a gradient asked for: the same
    assert torch.equal(ops.matmul(**args), got["out"])
    assert ops.check() == 0
    return args, dout, got


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("m,k", [(1, 8), (3, 72), (17, 264), (64, 1024), (200, 520), (300, 4096), (700, 200), (1030, 712)])
def test_one_matrix(m, k, activation):
    """From a token to tiles of CTA pairs, every activation, nothing else in the epilogue."""
    check(m, 512, k, activation=activation)


@pytest.mark.parametrize("n", [1, 3, 8, 33, 127, 129, 260, 1000])
@pytest.mark.parametrize("m", [2, 130, 1500])
def test_odd_columns(m, n):
    check(m, n, 136, activation="gelu", bias=F32, residual=True)


@pytest.mark.parametrize("dtype,out_dtype,bias", [(BF16, F32, BF16), (F16, F16, F32), (F16, F32, F16), (BF16, BF16, BF16)])
@pytest.mark.parametrize("activation,n", [("silu", 252), ("swiglu", 768)])
@pytest.mark.parametrize("m", [5, 1111])
def test_types(m, n, activation, dtype, out_dtype, bias):
    check(m, n, 328, activation=activation, bias=bias, residual=True, dtype=dtype, out_dtype=out_dtype)


GROUPS = [
    [0, 1, 31, 64, 0, 65, 200, 3, 17, 16],  # every kind of last block
    [0, 0, 0],
    [700],
    [5, -3, 1 << 30, 9],  # negative: none; more than there are: what is left
    [1] * 40,
]


@pytest.mark.parametrize("activation", [None, "swiglu", "gelu"])
@pytest.mark.parametrize("number", range(len(GROUPS)))
@pytest.mark.parametrize("spare", [0, 37])
def test_groups(number, activation, spare):
    groups = GROUPS[number]
    m = 90 if max(groups) > 1 << 20 else max(1, sum(groups)) + spare
    check(m, 512, 200, groups, activation, bias=F32, residual=number % 2 == 1)


@pytest.mark.parametrize("n,k,activation", [(1, 8, None), (77, 40, "relu"), (260, 1048, "silu")])
def test_groups_of_odd_sizes(n, k, activation):
    check(333, n, k, [100, 0, 7, 129, 64, 21], activation, bias=BF16, residual=True, out_dtype=F32)


@pytest.mark.parametrize("n,k", [(256, 64), (512, 128), (768, 320), (264, 192), (512, 200), (1024, 72)])
def test_weights_in_whole_chunks_and_others(n, k):
    """Operands that lie across the sum are loaded by chunks of 64 columns, two at a time where all are whole."""
    check(400, n, k, [15, 129, 0, 64, 1, 191])
    check(333, n, k)


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("groups", [None, [600, 1, 0, 99]])
def test_a_residual_in_16_bits(activation, groups):
    """Through shared memory on its way to the matrix fragments, or not, where its rows are off a boundary: the same bits."""
    args, dout, got = check(707, 512, 136, groups, activation, F32, True)
    wide = torch.zeros(708, args["residual"].shape[1] + 4, dtype=BF16, device="cuda")
    off = wide[1:, 4:]
    off.copy_(args["residual"])
    assert torch.equal(ops.matmul(**{**args, "residual": off}), got["out"])


def test_many_groups():
    g = torch.Generator().manual_seed(0)
    groups = torch.randint(0, 4, (1024,), generator=g).tolist()
    check(sum(groups) + 5, 72, 64, groups, bias=F32)


def test_a_group_of_many_tiles():
    check(5000, 768, 320, [4000, 3, 900], "swiglu")


@pytest.mark.parametrize("groups", [None, [40, 0, 23, 33]])
def test_neighbours_that_are_no_numbers(groups):
    """Nothing of another group, of rows behind the last, of padding around rows or of another matrix comes into a result."""
    args, dout = make_case(96, 264, 72, groups, "silu", F32, False, BF16, BF16, 5, "cuda")
    wide = torch.full((98, 128), float("nan"), dtype=BF16, device="cuda")
    wide[1:97, 8:80] = args["a"]
    rows = wide[1:97, 8:80]
    clean = run(args, dout)
    again = run({**args, "a": rows}, dout)
    for name in clean:
        assert torch.equal(clean[name], again[name]), name
    if groups is None:
        return
    # one group's rows and matrix are infinite: the other groups do not notice
    a, b = args["a"].clone(), args["b"].clone()
    a[40:63] = float("inf")
    b[2] = float("nan")
    b[1] = float("nan")  # of a group without rows
    bad = run({**args, "a": a, "b": b}, dout)
    for name in ("out", "da"):
        assert torch.equal(bad[name][:40], clean[name][:40]) and torch.equal(bad[name][63:], clean[name][63:])
    for name in ("db", "dbias"):
        for g in (0, 1, 3):
            assert torch.equal(bad[name][g], clean[name][g]), (name, g)
    assert not bad["db"][1].any() and not bad["dbias"][1].any()


@pytest.mark.parametrize("by,pad", [(1, 0), (8, 8), (3, 5), (4, 4)])
def test_rows_apart_and_off_a_boundary(by, pad):
    args, dout = make_case(150, 96, 72, None, "relu", F32, True, BF16, BF16, 2, "cuda")
    clean = run(args, dout)

    def moved(t):
        flat = torch.zeros(t.shape[0] * (t.shape[1] + pad) + by, dtype=t.dtype, device="cuda")
        view = flat[by:].view(t.shape[0], -1)[:, : t.shape[1]]
        view.copy_(t)
        return view

    a, residual, d = (moved(t).requires_grad_() for t in (args["a"], args["residual"], dout))
    out = ops.matmul(**{**args, "a": a, "residual": residual})
    assert torch.equal(out, clean["out"])
    da, dr = torch.autograd.grad(out, (a, residual), d.detach())
    assert torch.equal(da, clean["da"]) and torch.equal(dr, clean["dresidual"])
    # and transposed
    out = ops.matmul(**{**args, "a": args["a"].T.contiguous().T, "residual": args["residual"].T.contiguous().T})
    assert torch.equal(out, clean["out"])
    # a gradient whose rows are one row
    a = args["a"].clone().requires_grad_()
    plain = ops.matmul(a, args["b"])
    (da,) = torch.autograd.grad(plain, a, torch.ones(1, 1, dtype=BF16, device="cuda").expand(150, 96), retain_graph=True)
    assert torch.equal(da, torch.autograd.grad(plain, a, torch.ones(150, 96, dtype=BF16, device="cuda"))[0])


def test_no_rows():
    b = torch.randn(64, 32, device="cuda").bfloat16().requires_grad_()
    a = torch.empty(0, 32, dtype=BF16, device="cuda").requires_grad_()
    bias = torch.zeros(64, device="cuda").requires_grad_()
    out = ops.matmul(a, b, bias, "silu")
    assert out.shape == (0, 64)
    da, db, dbias = torch.autograd.grad(out, (a, b, bias), torch.empty_like(out))
    assert da.shape == (0, 32) and not db.any() and not dbias.any()


@pytest.mark.parametrize("groups", [None, [50, 0, 150, 100]])
def test_same_bits_every_time_and_one_gradient_at_a_time(groups):
    args, dout = make_case(300, 512, 264, groups, "gelu", F32, True, BF16, BF16, 4, "cuda")
    first = run(args, dout)
    for _ in range(3):
        for name, t in run(args, dout).items():
            assert torch.equal(t, first[name]), name
    for name in ("a", "b", "bias", "residual"):
        leaf = args[name].clone().requires_grad_()
        out = ops.matmul(**{**args, name: leaf})
        assert torch.equal(torch.autograd.grad(out, leaf, dout)[0], first["d" + name]), name


def test_offsets_behind_2_to_the_31():
    """A result of more than 2^31 values, and a sum over its rows."""
    m, n, k = 70_000, 32_768, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    a = torch.randn(m, k, device="cuda", generator=g).bfloat16()
    b = torch.randn(n, k, device="cuda", generator=g).bfloat16().requires_grad_()
    out = ops.matmul(a, b)
    assert out.numel() > 2**31
    rows = torch.tensor([0, 65_535, 65_536, 65_600, m - 1], device="cuda")
    want = a[rows].float() @ b.detach().float().T
    torch.testing.assert_close(out.detach()[rows].float(), want, rtol=2**-8, atol=2**-12 * 64)
    dout = torch.zeros_like(out)
    dout[-1] = 1
    (db,) = torch.autograd.grad(out, b, dout)
    assert torch.equal(db, a[-1].expand(n, k))


def test_a_long_sum():
    check(64, 128, 65_536)
    check(300, 256, 30_000)


def test_on_another_stream_and_captured():
    args, dout = make_case(400, 512, 264, [100, 0, 250, 30], "swiglu", F32, True, BF16, BF16, 8, "cuda")
    plain = run(args, dout)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = run(args, dout)
    torch.cuda.current_stream().wait_stream(stream)
    for name in plain:
        assert torch.equal(plain[name], other[name])
    leaves = {name: args[name].clone().requires_grad_() for name in ("a", "b", "bias", "residual")}

    def step():
        out = ops.matmul(**{**args, **leaves})
        return out.detach(), torch.autograd.grad(out, tuple(leaves.values()), dout)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = step()
    for seed in (1, 2):
        fresh, _ = make_case(400, 512, 264, [100, 0, 250, 30], "swiglu", F32, True, BF16, BF16, seed, "cuda")
        with torch.no_grad():
            for name, leaf in leaves.items():
                leaf.copy_(fresh[name])
            args["rows"].copy_(torch.tensor([[7, 300, 2, 1], [0, 0, 0, 399]][seed - 1], dtype=torch.int32))  # other groups, too
        graph.replay()
        torch.cuda.synchronize()
        now_out, now = step()
        assert torch.equal(out, now_out)
        for a, b in zip(grads, now):
            assert torch.equal(a, b)


def test_two_at_once():
    """Calls on several streams share nothing: each has the bits that it has alone."""
    cases = [make_case(m, 512, 264, groups, "silu", F32, False, BF16, BF16, m, "cuda") for m, groups in ((300, [100, 200]), (40, None), (900, None))]
    alone = [run(*case) for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    together = []
    for _ in range(5):
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                together.append(run(*case))
    torch.cuda.synchronize()
    for i, got in enumerate(together):
        for name, t in got.items():
            assert torch.equal(t, alone[i % len(cases)][name])


@pytest.mark.parametrize("number", range(22))
def test_refuses(number):
    changed, words = refusals("cuda")[number]
    good = {"a": torch.zeros(4, 16, dtype=BF16, device="cuda"), "b": torch.zeros(8, 16, dtype=BF16, device="cuda")}
    assert ops.matmul(**good).shape == (4, 8)
    with pytest.raises(ValueError, match=words):
        ops.matmul(**{**good, **changed})


def test_refuses_other_devices_and_weights_off_a_boundary():
    a, b = torch.zeros(4, 16, dtype=BF16, device="cuda"), torch.zeros(8, 16, dtype=BF16, device="cuda")
    for changed in ({"b": b.cpu()}, {"bias": torch.zeros(8)}, {"residual": torch.zeros(4, 8, dtype=BF16)}, {"rows": torch.zeros(1, dtype=torch.int32), "b": b[None]}):
        with pytest.raises(ValueError, match="device"):
            ops.matmul(**{"a": a, "b": b, **changed})
    with pytest.raises(ValueError, match="16-byte"):
        ops.matmul(a, torch.zeros(129, dtype=BF16, device="cuda")[1:].view(8, 16))


@pytest.mark.parametrize("through_leaf", [False, True])
def test_a_capture_beside_a_living_graph(through_leaf):
    """A leaf whose gradient is collected on the default stream, by a graph that still lives, is refused inside a capture; once that
    graph is gone, or where it hangs on no leaf of the call, the capture goes through."""
    a = torch.randn(32, 64, device="cuda").bfloat16().requires_grad_()
    b = torch.randn(64, 64, device="cuda").bfloat16().requires_grad_()
    living = ops.matmul(a, b)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still holds this leaf"):
        with torch.cuda.graph(graph):
            ops.matmul(a, b)
    del living
    dout = torch.ones(32, 64, device="cuda", dtype=BF16)
    other = ops.matmul(a.detach().clone().requires_grad_(), b.detach()) if through_leaf else None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        da, db = torch.autograd.grad(ops.matmul(a, b), (a, b), dout)
    graph.replay()
    want = torch.autograd.grad(ops.matmul(a, b), (a, b), dout)
    assert torch.equal(da, want[0]) and torch.equal(db, want[1])
    assert other is None or other.requires_grad
