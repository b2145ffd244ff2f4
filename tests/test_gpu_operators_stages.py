"""One MoE block through the operators, each step checked in 64 bits from the
values that the step itself was given, so that every term (the gate, a norm's
weights, the scale of the branch, a routing weight) is held to its roundings.

Tolerances, u = 2^-24: the products as in test_gpu_q4.py; the combine, one
fused multiply-add a choice, (top_k + 1) u of the absolute sum; the norms c = 96
as in test_gpu_norm_rows.py; a bf16 result half a step, 2^-8, more."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_operators_chain import Block  # noqa: E402
from test_gpu_q4 import ACTS, close, dense  # noqa: E402
from test_gpu_residual_norm import U, Bound, near, rms, up  # noqa: E402

EPS = float(np.float32(1e-6))


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


def check_stages(b):
    hidden = up(b.hidden)
    r = rms(hidden.v, EPS)
    near(b.rms_x, r, 96, "rms_x")
    near(b.x, hidden * r * up(b.w_pre), 96, "x")

    ids = b.ids.cpu().numpy()
    flat = ids.reshape(-1)
    order = sorted((a for a in range(flat.size) if flat[a] >= 0), key=lambda a: (flat[a], a))
    assert b.plan["perm"].cpu().tolist()[:len(order)] == order
    place = {a: p for p, a in enumerate(order)}
    assert b.plan["position"].cpu().tolist() == [place.get(a, -1) for a in range(flat.size)]

    x, h, rows = b.x.cpu().double(), b.h.cpu(), b.rows.cpu()
    experts = flat[order]
    for e in set(experts.tolist()):
        at = torch.as_tensor(np.nonzero(experts == e)[0])
        token = torch.as_tensor(np.asarray(order)[at.numpy()] // b.K)
        gate_up, down = (dense(b.codes[i][e].cpu(), b.scales[i][e].cpu(), None, "e2m1", 32) for i in range(2))
        close(h[at], gate_up, x[token], 32, act=ACTS[0])
        close(rows[at], down, h[at].double(), 32)

    y = Bound(torch.zeros(b.T, b.H, dtype=torch.float64))
    w = b.w.cpu().double()
    for t in range(b.T):
        for j in range(b.K):
            if t * b.K + j in place:
                term = w[t, j] * rows[place[t * b.K + j]].double()
                y.v[t] += term
                y.a[t] += term.abs()
    near(b.y, y, b.K + 1, "y")

    y = up(b.y)
    ry = rms(y.v, EPS)
    near(b.rms_y, ry, 96, "rms_y")
    out = hidden + Bound(torch.sigmoid(b.gate.cpu().double())[:, None]) * (y * ry * up(b.w_post)) * 0.5
    near(b.out, out, 96, "out")
    r = rms(out.v, EPS)
    # the root's error from out's: at most |d out| / |out| over the row
    grow = (out.a * out.a).sum(1, keepdim=True).sqrt() / (out.v * out.v).sum(1, keepdim=True).sqrt()
    rx = Bound(r.v, r.v * (1 + grow))
    near(b.rms_next, rx, 96, "rms_next")
    near(b.next_x, out * rx * up(b.w_next), 96, "next_x")


@pytest.mark.parametrize("T, K, E, H, I, drop", [
    (1, 4, 8, 256, 128, 0.0), (5, 2, 4, 512, 96, 0.0), (32, 4, 16, 320, 224, 0.2), (40, 8, 8, 1024, 160, 0.0),
    (24, 4, 60, 640, 544, 0.1),
])
def test_block(eng, L, T, K, E, H, I, drop):
    b = Block(L, eng, T, K, E, H, I, T)
    b.feed(T + 1, drop)
    b.ids[:, 0] = b.ids[:, 0].clamp(min=0)  # every token keeps one expert: RMSNorm of a zero y is eps' own
    b.run()
    eng.sync()
    check_stages(b)


def test_replayed_with_new_inputs(eng, L):
    b = Block(L, eng, 16, 4, 12, 512, 128, 1)
    b.feed(0)
    b.run()
    torch.cuda.synchronize()
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        b.run(torch.cuda.current_stream().cuda_stream)
    for seed in (3, 4):
        b.feed(seed)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_stages(b)
    eng.sync()
    del g


@pytest.mark.parametrize("change", ["no gate", "no scale", "no post_w", "no next_w", "no branch", "one choice less"])
def test_the_bounds_tell_a_missing_term(eng, L, change):
    """The outputs as they would be with a term left out do not pass."""
    b = Block(L, eng, 40, 8, 8, 1024, 160, 40)
    b.feed(41)
    b.run()
    eng.sync()
    check_stages(b)
    c = lambda t: t.cpu().double()  # noqa: E731
    y = c(b.y)
    n = y / torch.sqrt((y * y).mean(1, keepdim=True) + EPS) * (1.0 if change == "no post_w" else c(b.w_post))
    g = 1.0 if change == "no gate" else torch.sigmoid(c(b.gate))[:, None]
    out = c(b.hidden) + (0.0 if change == "no branch" else 1.0 if change == "no scale" else 0.5) * g * n
    nxt = out / torch.sqrt((out * out).mean(1, keepdim=True) + EPS) * (1.0 if change == "no next_w" else c(b.w_next))
    if change == "one choice less":
        pos = b.plan["position"].cpu().long().view(b.T, b.K)
        b.y -= (b.w.cpu()[:, -1:] * b.rows.cpu()[pos[:, -1]]).cuda()
    elif change == "no next_w":
        b.next_x.copy_(nxt)
    else:
        b.out.copy_(out)
    with pytest.raises(AssertionError):
        check_stages(b)
    if change not in ("one choice less", "no next_w"):  # and the next block's input by itself
        b.run()
        eng.sync()
        b.next_x.copy_(nxt)
        with pytest.raises(AssertionError):
            check_stages(b)
