"""The norms and their gradients with more rows than a block's ring holds at
once, so that its places are filled again and the waits change their phase,
and the lengths at which another kernel takes over.

Tolerances are those of test_gpu_residual_norm.py, of values as the kernels
form them now:
  * forward, sums over a row in fp32: a thread adds up at most 32 squares, the
    lanes 5 steps, the warps 6 (by fours, 16 of them): 43, of which the root
    halves the relative error; fewer than 40 roundings around it: c = 96.
  * gradients, rows: three sums, of at most 64 terms a thread (rows above 8192
    columns), 5 steps over the lanes and 8 over the warps, below 85, and fewer
    than 30 roundings around: c = 128.
  * sums over the tokens: a block adds at most ceil(T / 148) rows, the last
    kernel at most 14 of its 444 blocks one after the other and 5 steps over
    the lanes, each term with a row's error of 128: below 176 + T / 148."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_residual_norm import (check_backward, forward_reference, make, near, roots, run_backward,  # noqa: E402
                                    run_forward)


@pytest.fixture(scope="module")
def L(pkg):
    import moe_b200.lib as lib
    return lib


@pytest.fixture(scope="module")
def eng(L):
    e = L.Engine(0)
    yield e
    e.sync()
    e.close()


# T, H, types of hidden / y / x, gate, sigmoid, post, pre, unit offset, residual scale, out scale, extra columns
REST = (True, True, False, 1.0, 1.0, 0)  # both norms, scales of 1, rows back to back
BOTH = [
    # 444 blocks of 256 threads, two stages: five or six rows a block
    (2311, 2048, "bf16", "bf16", "bf16", "element", True) + REST,
    (2311, 2048, "f32", "bf16", "bf16", "channel", False) + REST,
    (2311, 2048, "bf16", "f32", "f32", "token", True, True, True, True, 0.75, -0.5, 8),
    # 3552 blocks of a warp
    (18100, 64, "f32", "bf16", "bf16", "token", True) + REST,
    # 296 blocks of 384 threads and 148 of 512, whose weights stay in registers
    (1411, 2880, "f32", "f32", "bf16", "none", False) + REST,
    (1411, 2880, "bf16", "bf16", "bf16", "element", False) + REST,
    (1111, 4096, "bf16", "bf16", "bf16", "channel", True) + REST,
    (1111, 4096, "f32", "bf16", "bf16", "element", True) + REST,
    # 148 blocks of up to 1024 threads
    (701, 7168, "f32", "bf16", "bf16", "channel", False, True, True, False, 1.0, 0.5, 0),
    (701, 7168, "bf16", "bf16", "bf16", "token", True) + REST,
    (701, 5632, "bf16", "bf16", "bf16", "element", True) + REST,
    # rows that do not fit the ring
    (451, 8192, "f32", "f32", "f32", "channel", True) + REST,
    (451, 12288, "bf16", "bf16", "bf16", "element", True) + REST,
    # rows that cannot be read by vectors: 444 blocks, 148, 148 with rows read twice
    (1511, 2043, "bf16", "bf16", "bf16", "element", True) + REST,
    (1511, 2043, "f32", "bf16", "bf16", "token", False) + REST,
    (331, 5001, "f32", "bf16", "bf16", "channel", True) + REST,
    (331, 5001, "bf16", "bf16", "bf16", "none", False) + REST,
    (331, 5001, "bf16", "f32", "bf16", "element", True) + REST,
    (331, 9001, "f32", "bf16", "bf16", "channel", False) + REST,
]


@pytest.mark.parametrize("case", BOTH)
def test_gradients_of_many_rows(eng, L, case):
    d = make(case)
    ry, rx = roots(d, case)
    check_backward(run_backward(eng, L, d, case, ry, rx), d, case, ry, rx)


@pytest.mark.parametrize("case", [BOTH[0], BOTH[4], BOTH[9], BOTH[13]])
@pytest.mark.parametrize("without", ["d_hidden_out", "d_x"])
def test_gradients_of_many_rows_with_one_coming_in(eng, L, case, without):
    d = make(case)
    d[without] = None
    ry, rx = roots(d, case)
    check_backward(run_backward(eng, L, d, case, ry, rx if without != "d_x" else None), d, case, ry, rx)


@pytest.mark.parametrize("case", [
    (2311, 2048, "bf16", "bf16", "bf16", "channel", True, False, True, False, 1.0, 1.0, 0),   # no norm behind
    (701, 7168, "f32", "bf16", "bf16", "none", False, True, False, False, 1.0, 1.0, 0),       # only the add
    (1411, 4096, "f32", "f32", "bf16", None, False, False, True, True, 1.0, 1.0, 0),          # only the norm in front
    (1511, 2043, "bf16", "bf16", "f32", None, False, False, True, False, 1.0, 1.0, 0),
])
def test_gradients_of_part_of_the_edge(eng, L, case):
    d = make(case)
    ry, rx = roots(d, case)
    check_backward(run_backward(eng, L, d, case, ry, rx), d, case, ry, rx)


@pytest.mark.parametrize("case", [BOTH[0], BOTH[6], BOTH[9], BOTH[12], BOTH[13]])
def test_gradients_of_many_rows_in_place(eng, L, case):
    """Over the gradient that came in and over y, and some of them alone: the same bits."""
    d = make(case)
    ry, rx = roots(d, case)
    apart = run_backward(eng, L, d, case, ry, rx)
    d2 = {k: None if v is None else v.clone() for k, v in d.items()}
    got = run_backward(eng, L, d2, case, ry, rx, d_hidden=d2["d_hidden_out"], d_y=d2["y"])
    some = run_backward(eng, L, d, case, ry, rx, ("d_y", "d_pre_w"))
    for k, v in apart.items():
        assert v is None or torch.equal(v, got[k]), k
        assert some[k] is None or torch.equal(v, some[k]), k


FORWARD = [
    (9, 7168, "f32", "bf16", "bf16", "channel", False, True, True, False, 1.0, 0.5, 0),
    (5, 16384, "bf16", "bf16", "bf16", "element", True) + REST,
    (5, 9000, "f32", "bf16", "bf16", "token", True) + REST,
    (7, 4097, "bf16", "bf16", "bf16", "element", True) + REST,
    (7, 5001, "f32", "bf16", "bf16", "channel", True) + REST,
    (5, 8193, "f32", "f32", "bf16", "none", False) + REST,
    (3, 16383, "bf16", "bf16", "bf16", "channel", False) + REST,
    (6, 5001, "f32", "f32", "bf16", None, False, False, True, False, 1.0, 1.0, 0),
    (3000, 256, "bf16", "bf16", "bf16", "element", True) + REST,
    (3001, 264, "f32", "bf16", "bf16", "channel", True) + REST,
]


@pytest.mark.parametrize("case", FORWARD)
def test_forward_lengths(eng, L, case):
    d = make(case)
    got = run_forward(eng, L, d, case)
    for k, want in forward_reference(d, case).items():
        near(got[k], want, 96, k)
