"""The operators' entry points with what a caller may hand them by mistake:
configs that no call takes, tensors of another element type, calls from two
threads.  Without a GPU, like test_operators_cpu.py."""
import subprocess
import sys
import threading
from pathlib import Path

import pytest

from test_operators_cpu import FakeTensor


@pytest.fixture(scope="module")
def L(pkg):
    import moe_b200.build as build
    import moe_b200.lib as lib
    build.build()
    lib.load()
    return lib


QUERY = """
import sys
import threading
sys.path.insert(0, sys.argv[1])
import conftest
conftest.load_pkg()
import moe_b200.lib as L
make, size = L.Engine.residual_norm_cfg, L.Engine.residual_norm_workspace_bytes
bad = [make(h, 16) for h in (0, 32769, 2 ** 32 - 255, 2 ** 32 - 1)]
bad += [make(64, 1 << 31), make(64, 16, gate=4), make(64, 16, y_type=2), make(64, 16, y_stride=63)]
print([size(c) for c in bad], size(None))
print(size(make(1, 16)), size(make(32768, 200)))
"""


def test_workspace_query_of_configs_that_no_call_takes(L):
    """The query comes before the call that refuses the config: it answers 0 and
    lives.  In a process of its own, which a division by zero would end."""
    r = subprocess.run([sys.executable, "-c", QUERY, str(Path(__file__).parent)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    assert r.stdout.splitlines() == [f"{[0] * 8} 0", f"{16 * 2 * 4} {148 * 2 * 32768 * 4}"]


class Library:
    """Takes every call and says yes; `on` maps entry points to what they do instead."""

    def __init__(self, **on):
        self.on, self.calls = on, []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return self.on[name](*args) if name in self.on else 1
        return call


@pytest.fixture
def face(L, monkeypatch):
    def make(**on):
        lib = Library(**on)
        monkeypatch.setattr(L, "load", lambda: lib)
        eng = L.Engine(0)
        lib.calls.clear()
        return eng, lib
    return make


def tensor(shape, dtype):
    size = {"torch.float32": 4, "torch.int32": 4, "torch.uint32": 4, "torch.bfloat16": 2, "torch.float16": 2,
            "torch.int16": 2, "torch.int64": 8}.get(dtype, 1)
    return FakeTensor(shape, dtype, size)


F32, BF16, F16, I32, U32, U8, I8 = (f"torch.{t}" for t in (
    "float32", "bfloat16", "float16", "int32", "uint32", "uint8", "int8"))


def operands(L, fn):
    """Arguments of one good call: name -> (shape, element type, other types that are refused)."""
    P, T, K, E, H = 32, 16, 2, 8, 64
    index = {"perm": (P,), "offset": (E + 1,), "batches": (E, 4), "batch_count": (1,)}
    by_choice = {"position": ((P,), I32, [F32, U32]), "w": ((P,), F32, [I32])}
    if fn == "sort_tokens":
        return (T, K, E), dict(ids=((P,), I32, [F32, U32]), position=by_choice["position"],
                               **{k: (v, I32, [F32]) for k, v in index.items()})
    if fn in ("dispatch_rows", "dispatch_rows_backward", "combine_rows", "combine_rows_backward"):
        rows = {"dispatch_rows": ["x", "sorted"], "dispatch_rows_backward": ["d_sorted", "d_x"],
                "combine_rows": ["sorted", "y"], "combine_rows_backward": ["d_y", "sorted"]}[fn]
        out = {k: ((P if "sorted" in k else T, H), BF16, [F16, F32]) for k in rows}
        out["position"] = by_choice["position"]
        if "combine" in fn:
            out["w"] = by_choice["w"]
        if fn == "combine_rows_backward":
            out["d_w"] = ((P,), F32, [I32])
        return (L.Engine.rows_cfg(H, T, K, P),), out
    if fn in ("residual_norm", "residual_norm_backward"):
        cfg = L.Engine.residual_norm_cfg(H, T, gate=L.GATE_TOKEN)
        vec, per = ((H,), F32, [I32]), ((T,), F32, [I32])
        out = dict(post_w=vec, pre_w=vec, gate=per, rms_y=per, rms_x=per, y=((T, H), F32, [I32]))
        if fn == "residual_norm":
            out.update(hidden=((T, H), F32, [I32]))
        else:
            out.update(d_post_w=vec, d_pre_w=vec, d_gate=per)
        return (cfg,), out
    scale = {"q4_e8m0": (L.DTYPE_E8M0, U8, [I8]), "q4_bf16": (L.DTYPE_BF16, BF16, [F16, "torch.int16"]),
             "q4_f16": (L.DTYPE_F16, F16, [BF16]), "q4_f32": (L.DTYPE_F32, F32, [I32])}[fn]
    code = L.Q4_E2M1 if scale[0] == L.DTYPE_E8M0 else L.Q4_INT4
    cfg = L.Engine.q4_cfg(48, H, T, P, code=code, scale_type=scale[0], experts=E, top_k=K)
    out = dict(codes=((E, 48, H // 2), U8, ["torch.float8_e4m3fn"]), scales=((E, 48, 2), *scale[1:]),
               x=((T, H), BF16, [F16]), y=((P, 48), F32, [I32]),
               **{k: (index[k], U32, [F32]) for k in ("perm", "batches", "batch_count")})
    if code == L.Q4_INT4:
        out["zeros"] = ((E, 48, 2), U8, [I8])
    return (cfg,), out


@pytest.mark.parametrize("fn", ["sort_tokens", "dispatch_rows", "dispatch_rows_backward", "combine_rows",
                                "combine_rows_backward", "residual_norm", "residual_norm_backward", "q4_e8m0",
                                "q4_bf16", "q4_f16", "q4_f32"])
def test_element_types_are_those_of_the_config(L, face, fn):
    """A tensor of another type of the same size is refused by its name, and nothing runs."""
    eng, lib = face()
    method = "q4_matvec" if fn.startswith("q4") else fn
    entry = {"residual_norm": "moe_b200_residual_norm_forward"}.get(fn, f"moe_b200_{method}")
    first, ops = operands(L, fn)

    def call(**change):
        args = {k: tensor(shape, change.get(k, kind)) for k, (shape, kind, _) in ops.items()}
        if fn == "sort_tokens":
            eng.sort_tokens(args.pop("ids"), *first, **args)
        else:
            getattr(eng, method)(*first, **args)
    call()
    assert lib.calls == [entry]
    lib.calls.clear()
    for name, (_, _, others) in ops.items():
        for other in others:
            with pytest.raises(L.MoEError, match=rf"^{name}\b.*{other}"):
                call(**{name: other})
    assert not lib.calls


def test_types_with_the_same_meaning_are_taken(L, face):
    eng, lib = face()
    t = tensor
    cfg = L.Engine.q4_cfg(48, 64, 4)
    for codes in (U8, I8, "torch.float4_e2m1fn_x2"):
        for scales in (U8, "torch.float8_e8m0fnu"):
            eng.q4_matvec(cfg, t((48, 32), codes), t((48, 2), scales), t((4, 64), BF16), t((4, 48), F32))
    eng.sort_tokens(t((8,), I32), 4, 2, 8, position=t((8,), I32), perm=t((8,), U32), offset=t((9,), U32),
                    batches=t((8, 4), U32), batch_count=t((1,), U32))
    assert len(lib.calls) == 7


def test_refusals_of_two_threads_keep_their_messages(L, face):
    """Two calls of one engine refused at once: neither returns before both have
    written their messages, and each thread's error is its own."""
    both = threading.Barrier(2, timeout=30)

    def refuse(engine, stream, err):
        err.value = b"stream %d" % stream
        both.wait()
        return 0
    eng, _ = face(moe_b200_sync=refuse)
    said = {}

    def work(stream):
        try:
            eng.sync(stream)
        except L.MoEError as e:
            said[stream] = str(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in (1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert said == {1: "stream 1", 2: "stream 2"}


@pytest.mark.parametrize("name", ["residual_scale", "out_scale"])
def test_scales_of_zero_are_refused(L, name):
    """A zero (or what becomes one in fp32) would stand for 1 in the C config."""
    for value in (0.0, -0.0, 1e-50):
        with pytest.raises(L.MoEError, match=name):
            L.Engine.residual_norm_cfg(64, 4, **{name: value})
    for value in (1.0, -0.5, 1e-40):
        assert getattr(L.Engine.residual_norm_cfg(64, 4, **{name: value}), name) != 0.0


def test_products_by_expert_take_out_rows_as_it_is(L, face):
    """A rank to which no row was routed has an empty y, whatever the tokens; a
    config without out_rows for a y that has rows would leave them unwritten."""
    eng, lib = face()
    by = dict(batches=tensor((8, 4), I32), batch_count=tensor((1,), I32), perm=tensor((32,), I32))
    args = tensor((8, 48, 32), U8), tensor((8, 48, 2), U8), tensor((16, 64), BF16)
    cfg = L.Engine.q4_cfg(48, 64, 16, 0, experts=8, top_k=2)
    eng.q4_matvec(cfg, *args, tensor((0, 48), F32), **by)
    assert len(lib.calls) == 1
    with pytest.raises(L.MoEError, match="out_rows=0 .* y of 32 rows"):
        eng.q4_matvec(cfg, *args, tensor((32, 48), F32), **by)
    assert len(lib.calls) == 1
    eng.q4_matvec(L.Engine.q4_cfg(48, 64, 16, 32, experts=8, top_k=2), *args, tensor((32, 48), F32), **by)
    # without batches 0 stands for the tokens
    eng.q4_matvec(L.Engine.q4_cfg(48, 64, 16), tensor((48, 32), U8), tensor((48, 2), U8), args[2],
                  tensor((16, 48), F32))
    assert len(lib.calls) == 3
