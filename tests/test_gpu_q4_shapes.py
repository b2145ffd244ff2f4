"""4-bit products of large matrices against 64-bit products: the launch shapes
that a matrix only meets from a few blocks an SM on.  With 148 SMs:
  * four tiles of rows a block (a ring of two stages; gated: two tiles of gate
    and two of up rows) from 592 blocks of 64 outputs (32 gated) on, with up
    to 8 columns (8 bf16 rows, 2 fp32 rows);
  * four warps a block, or two with four tiles of columns (17 to 32 bf16
    rows), from 444 blocks on.
Outputs that are no multiple of a block's, columns that end inside a slice of
128 and give a block's warps different numbers of slices.  Tolerances are those
of test_gpu_q4.py: how a block is cut changes the order of a path's sums, of
which there are at most 128 terms of a slice, the slices and 16 warps, below
the 2 * (group + cols / group + 32) that are counted there."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_q4 import ACTS, DT, close, dense, kinds, weights  # noqa: E402


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


# tokens, N, K, code, group, scale, zeros, x, y, extra columns of x and y
DENSE = [
    # four tiles of rows
    (4, 37921, 1152, "int4", 128, "bf16", "yes", "bf16", "f32", 0),
    (1, 38001, 1056, "e2m1", 32, "e8m0", None, "bf16", "bf16", 8),
    (2, 37889, 1056, "e2m1", 32, "e8m0", None, "f32", "f32", 0),
    (8, 38001, 96, "int4", 32, "f16", "wide", "bf16", "f32", 0),
    (1, 37940, 1088, "e2m1", 64, "bf16", None, "f32", "f32", 0),
    (10, 37900, 544, "int4", 32, "f32", None, "bf16", "f32", 0),   # 9 to 16 rows: two tiles of columns
    # two warps with four tiles of columns, four warps with two and with one a term
    (32, 14209, 1056, "e2m1", 32, "e8m0", None, "bf16", "f32", 0),
    (41, 14300, 640, "int4", 128, "bf16", "yes", "bf16", "bf16", 0),
    (12, 14300, 1056, "int4", 32, "e8m0", None, "bf16", "f32", 0),
    (9, 14300, 1056, "e2m1", 32, "e8m0", None, "f32", "f32", 0),
    (16, 14211, 576, "int4", 64, "f16", "yes", "f32", "f32", 0),
    # two tiles of rows, four warps, rows of x that cannot be read by vectors
    (3, 14300, 544, "e2m1", 32, "e8m0", None, "bf16", "f32", 1),
]


@pytest.mark.parametrize("case", DENSE)
def test_dense(eng, L, case):
    T, N, K, code, group, scale, zeros, xt, yt, extra = case
    codes, scales, z = weights(T + N, 1, N, K, code, group, scale, zeros)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(T, K + extra, generator=g).to(DT[xt]).cuda()
    y = torch.full((T, N + extra), 5.0, dtype=DT[yt], device="cuda")
    k = kinds(L)
    cfg = L.Engine.q4_cfg(N, K, T, code=L.Q4_E2M1 if code == "e2m1" else L.Q4_INT4, group=group, scale_type=k[scale],
                          x_type=k[xt], y_type=k[yt], x_stride=K + extra, y_stride=N + extra)
    eng.q4_matvec(cfg, codes.cuda(), scales.cuda(), x[:, :K], y[:, :N], zeros=None if z is None else z.cuda())
    eng.sync()
    xs, y = x[:, :K].cpu().double(), y.cpu()
    for lo in range(0, N, 8192):
        rows = slice(lo, min(N, lo + 8192))
        w = dense(codes[:, rows], scales[:, rows], None if z is None else z[:, rows], code, group)[0]
        close(y[:, rows], w, xs, group)
    assert (y[:, N:] == 5.0).all()


# tokens, top_k, experts, N, K, code, group, scale, zeros, x, y, gated, activation, dropped
EXPERTS = [
    # four tiles of rows: 60 batches of one or two rows by 10 blocks of 32 gated outputs, by 16 of 64
    (16, 4, 60, 300, 1056, "e2m1", 32, "e8m0", None, "bf16", "f32", True, 0, 0.0),
    (16, 4, 60, 300, 1056, "e2m1", 32, "e8m0", None, "f32", "bf16", True, 1, 0.1),
    (16, 4, 60, 333, 640, "int4", 128, "bf16", "yes", "bf16", "f32", True, 2, 0.0),
    (16, 4, 60, 1000, 544, "int4", 32, "f16", "yes", "f32", "f32", False, 0, 0.0),
    # four warps: an average of 4 fp32 rows; two warps: of 18 bf16 rows
    (64, 4, 64, 300, 544, "e2m1", 32, "e8m0", None, "f32", "f32", False, 0, 0.0),
    (96, 6, 32, 250, 544, "e2m1", 32, "e8m0", None, "bf16", "f32", True, 0, 0.2),
]


@pytest.mark.parametrize("case", EXPERTS)
@pytest.mark.parametrize("skewed", [False, True])
def test_by_expert(eng, L, case, skewed):
    """`skewed`: every token has the first expert among its choices, so one batch has far more rows than the average
    by which the launch goes."""
    T, top, E, N, K, code, group, scale, zeros, xt, yt, gated, act, drop = case
    rng = np.random.default_rng(T + N)
    ids = np.stack([rng.choice(np.arange(1, E), top, replace=False) if skewed else rng.choice(E, top, replace=False)
                    for _ in range(T)]).astype(np.int32)
    if skewed:
        ids[:, 0] = 0
    else:  # every expert has a token, so that there are as many batches as can be
        ids.reshape(-1)[:E] = np.arange(E)
    ids[rng.random((T, top)) < drop] = -1
    P = T * top
    i32 = dict(dtype=torch.int32, device="cuda")
    plan = dict(position=torch.zeros(P, **i32), perm=torch.zeros(P, **i32), offset=torch.zeros(E + 1, **i32),
                batches=torch.zeros(min(E, P), 4, **i32), batch_count=torch.zeros(1, **i32))
    eng.sort_tokens(torch.as_tensor(ids).cuda(), T, top, E, **plan)
    codes, scales, z = weights(T, E, N * (2 if gated else 1), K, code, group, scale, zeros)
    g = torch.Generator().manual_seed(7)
    x = torch.randn(T, K, generator=g).to(DT[xt]).cuda()
    y = torch.full((P, N), 5.0, dtype=DT[yt], device="cuda")
    k = kinds(L)
    cfg = L.Engine.q4_cfg(N, K, T, P, L.Q4_E2M1 if code == "e2m1" else L.Q4_INT4, group, k[scale], E, top, k[xt],
                          k[yt], gated, act)
    eng.q4_matvec(cfg, codes.cuda(), scales.cuda(), x, y, zeros=None if z is None else z.cuda(),
                  batches=plan["batches"], batch_count=plan["batch_count"], perm=plan["perm"])
    eng.sync()
    offset, perm, xs, y = plan["offset"].cpu(), plan["perm"].cpu().long(), x.cpu().double(), y.cpu()
    for e in range(E):
        at = torch.arange(int(offset[e]), int(offset[e + 1]))
        if len(at):
            w = dense(codes[e], scales[e], None if z is None else z[e], code, group)
            close(y[at], w, xs[perm[at] // top], group, act=ACTS[act] if gated else None)
    assert (y[int(offset[E]):] == 5.0).all()
