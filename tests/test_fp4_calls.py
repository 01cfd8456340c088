"""The compiled binding of the 4-bit calls (csrc/fp4_calls.cpp) against the wrappers' own checks.

A call that the binding takes does what the wrapper would have done; what it
does not take is left to the wrapper untouched, so errors are the wrapper's.
"""

import pytest
import torch

from nano_vllm_ascend_b200 import ops_fp4

D, H, KVH, BS, NB, T = 128, 8, 2, 32, 6, 5
TAKEN = {"append": "_append", "read": "_read", "norm": "_norm_rope_append", "decode": "_decode",
         "prefill": "_prefill"}


def state(dev, pool_fill=0):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)
    i = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=dev)
    st = dict(pool=torch.zeros(ops_fp4.pool_shape(NB, BS, KVH), dtype=torch.uint8, device=dev), q=r(T, H, D),
              k=r(T, KVH, D), v=r(T, KVH, D), slots=i([3, 40, 170, 0, 99], torch.int64), wq=r(D), wk=r(D),
              cos=torch.randn(64, D, generator=g).to(dev), sin=torch.randn(64, D, generator=g).to(dev),
              pos=i([1, 5, 63, 0, 7], torch.int64), table=i([[5, 1], [0, 3], [2, 4], [1, 0], [3, 5]]),
              lens=i([64, 33, 1, 0, 40]), cu=i([0, 1, 2, 3, 4, 5]), err=i([0]), scale=0.1, ks=0.5, vs=2.0, max_q=1)
    st["out"] = torch.zeros_like(st["q"])
    st["ws"] = torch.zeros(1 << 22, dtype=torch.uint8, device=dev)
    return st


def run(op, st):
    if op == "append":
        ops_fp4.kv_append_fp4(st["pool"], st["k"], st["v"], st["slots"], st["ks"], st["vs"], st["err"])
        return [st["pool"], st["err"]]
    if op == "read":
        return [*ops_fp4.kv_read_fp4(st["pool"], st["slots"], st["ks"], st["vs"], st.get("dtype", torch.bfloat16),
                                     error_word=st["err"]), st["err"]]
    if op == "norm":
        q = ops_fp4.qk_norm_rope_append_fp4(st["q"], st["k"], st["v"], st["wq"], st["wk"], 1e-6, st["cos"], st["sin"],
                                            st["pos"], st["pool"], st["slots"], st["ks"], st["vs"], st.get("q_out"),
                                            st["err"])
        return [q, st["pool"], st["err"]]
    if op == "decode":
        out = ops_fp4.paged_decode_fp4(st["out"], st["q"], st["pool"], st["table"], st["lens"], st["scale"], st["ws"],
                                       st.get("ctas", 0), st["ks"], st["vs"])
        assert out is st["out"]
        return [out, st["ws"][:4]]
    out = ops_fp4.paged_prefill_fp4(st["out"], st["q"], st["pool"], st["table"], st["cu"], st["lens"], st["max_q"],
                                    st["scale"], st["ks"], st["vs"], st["err"])
    assert out is st["out"]
    return [out, st["err"]]


@pytest.mark.gpu
@pytest.mark.parametrize("op,change", [
    ("append", {}), ("append", dict(err=None)), ("append", dict(ks=1, vs=2)), ("append", dict(slots=[3, 192, -1, 0, 9])),
    ("read", {}), ("read", dict(dtype=torch.float16)), ("read", dict(slots=[3, 192, -1, 0, 0])), ("norm", {}),
    ("norm", dict(q_out=True)), ("norm", dict(pos=[1, 64, -1, 0, 7])), ("decode", {}), ("decode", dict(ctas=3)),
    ("decode", dict(lens=[64, 65, 1, 0, 40])), ("prefill", {}), ("prefill", dict(lens=[64, 65, 1, 0, 40]))])
def test_a_call_that_is_taken_does_what_the_wrapper_does(cuda_device, monkeypatch, op, change):
    """The same bits both ways (filled pools, bad slots, positions and lengths with their error bits among them)."""
    assert ops_fp4._calls is not None, "the binding is built with the library"
    results = []
    for taken in (True, False):
        st = state(cuda_device)
        run("append", dict(st, slots=torch.arange(NB * BS, device=cuda_device),
                           k=torch.randn(NB * BS, KVH, D, generator=torch.Generator(cuda_device).manual_seed(3),
                                         device=cuda_device).to(torch.bfloat16),
                           v=torch.randn(NB * BS, KVH, D, generator=torch.Generator(cuda_device).manual_seed(4),
                                         device=cuda_device).to(torch.float16).to(torch.bfloat16)))
        for key, value in change.items():
            if isinstance(value, list):
                value = torch.tensor(value, dtype=st[key].dtype, device=cuda_device)
            st[key] = torch.full_like(st["q"], 7) if key == "q_out" else value
        seen = []
        with monkeypatch.context() as m:
            if taken:
                fast = getattr(ops_fp4, TAKEN[op])
                m.setattr(ops_fp4, TAKEN[op], lambda *a: seen.append(fast(*a)) or seen[-1])
            else:
                m.setattr(ops_fp4, TAKEN[op], ops_fp4._leave)
            results.append([t.clone() for t in run(op, st) if t is not None])
        assert not taken or (seen and not (seen[0].__class__ is int and seen[0] == ops_fp4._NOT_TAKEN))
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def bad(dev):
    """(operator, what a caller gives wrong): what only the binding could let through."""
    f = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=dev)
    yield "append", dict(k=f(T, KVH, D, t=torch.float32))
    yield "append", dict(k=f(T, KVH, D), v=f(T, KVH, D, t=torch.float16))
    yield "append", dict(k=f(T, KVH, 64), v=f(T, KVH, 64))
    yield "append", dict(k=f(T, KVH + 1, D), v=f(T, KVH + 1, D))
    yield "append", dict(v=f(T + 1, KVH, D))
    yield "append", dict(slots=f(T, t=torch.int32))
    yield "append", dict(slots=f(T + 1, t=torch.int64))
    yield "append", dict(k=f(KVH, T, D).transpose(0, 1), v=f(KVH, T, D).transpose(0, 1))
    yield "append", dict(err=f(1, t=torch.int64))
    yield "append", dict(err=f(0, t=torch.int32))
    yield "append", dict(ks=3.0)
    yield "append", dict(pool=f(NB, KVH, BS // 16, 2303, t=torch.uint8))
    yield "append", dict(pool=f(NB, BS // 16, KVH, 2304, t=torch.uint8).transpose(1, 2))
    yield "append", dict(pool=f(NB, KVH, 3, 2304, t=torch.uint8))
    yield "append", dict(k=torch.zeros(T, KVH, D, dtype=torch.bfloat16))
    yield "read", dict(slots=f(T, t=torch.int32))
    yield "read", dict(pool=f(NB, KVH, BS // 16, 2304, t=torch.int8))
    yield "read", dict(dtype=torch.float32)
    yield "read", dict(vs=0.0)
    yield "norm", dict(q=f(T, H, D, t=torch.float16))
    yield "norm", dict(q=f(T - 1, H, D))
    yield "norm", dict(wq=f(D, t=torch.float32))
    yield "norm", dict(wk=f(2 * D)[::2])
    yield "norm", dict(cos=f(64, 64, t=torch.float32))
    yield "norm", dict(sin=f(65, D, t=torch.float32))
    yield "norm", dict(sin=f(64, 2 * D, t=torch.float32)[:, ::2])
    yield "norm", dict(pos=f(T, t=torch.int32))
    yield "norm", dict(q_out=f(T, H, D, t=torch.float32))
    yield "norm", dict(q_out=f(T, H + 1, D))
    yield "decode", dict(out=f(T, H, D, t=torch.float32))
    yield "decode", dict(q=f(T, H, 2 * D)[:, :, ::2])
    yield "decode", dict(table=f(T, 2, t=torch.int64))
    yield "decode", dict(table=f(2, T, t=torch.int32).t())
    yield "decode", dict(table=f(1, 2, t=torch.int32).expand(T, 2))
    yield "decode", dict(lens=f(T + 1, t=torch.int32))
    yield "decode", dict(lens=f(2 * T, t=torch.int32)[::2])
    yield "decode", dict(table=f(T + 1, 2, t=torch.int32), lens=f(T + 1, t=torch.int32))
    yield "decode", dict(ws=f(64, t=torch.uint8))
    yield "decode", dict(scale=0.0)
    yield "decode", dict(scale=float("nan"))
    yield "decode", dict(ctas=-1)
    yield "decode", dict(q=f(T, 18, D), out=f(T, 18, D))
    yield "prefill", dict(cu=f(T, t=torch.int32))
    yield "prefill", dict(cu=f(T + 1, t=torch.int64))
    yield "prefill", dict(max_q=-1)
    yield "prefill", dict(scale=-1.0)
    yield "prefill", dict(q=f(T, 7, D), out=f(T, 7, D))


@pytest.mark.gpu
def test_what_is_wrong_is_refused_as_by_the_wrapper(cuda_device, monkeypatch):
    for op, change in bad(cuda_device):
        messages = []
        for taken in (True, False):
            st = dict(state(cuda_device), **change)
            with monkeypatch.context() as m:
                if not taken:
                    m.setattr(ops_fp4, TAKEN[op], ops_fp4._leave)
                with pytest.raises((ValueError, RuntimeError)) as e:
                    run(op, st)
            messages.append((e.type, str(e.value)))
            for name in ("pool", "out", "ws"):
                assert not st[name].any(), (op, change.keys(), "nothing was launched")
        assert messages[0] == messages[1], (op, list(change))


@pytest.mark.gpu
def test_repairable_arguments_are_repaired(cuda_device):
    """Index tensors that are strided are copied by the wrapper, as before; numbers may be numpy's."""
    import numpy as np

    st = state(cuda_device)
    want = [t.clone() for t in run("norm", st)]
    again = state(cuda_device)
    for name in ("slots", "pos"):
        wide = torch.zeros(2 * T, dtype=torch.int64, device=cuda_device)
        wide[::2] = again[name]
        again[name] = wide[::2]
    again["ks"] = np.float64(again["ks"])
    for a, b in zip(run("norm", again), want):
        assert torch.equal(a, b)


def test_host_tensors_are_left_to_the_wrapper():
    if ops_fp4._calls is None:
        pytest.skip("the binding is not built")
    st = state("cpu")
    c = ops_fp4._calls
    assert c.NOT_TAKEN == ops_fp4._NOT_TAKEN
    assert c.append(st["pool"], st["k"], st["v"], st["slots"], 1.0, 1.0, None) == c.NOT_TAKEN
    assert c.read(st["pool"], st["slots"], 1.0, 1.0, False, None) == c.NOT_TAKEN
    assert c.append(None, 1, "x", st["slots"], 1.0, 1.0, None) == c.NOT_TAKEN
    with pytest.raises(TypeError, match="3 arguments, 7 expected"):
        c.append(1, 2, 3)
    with pytest.raises(ValueError, match="must be a CUDA tensor|CUDA"):
        run("append", st)


@pytest.mark.gpu
def test_captured_calls_allocate_in_the_graph(cuda_device):
    """Outputs that a captured call allocates belong to the graph; a replay on new inputs writes them again."""
    st = state(cuda_device)
    st["err"] = None
    want = []
    for seed in (0, 1):
        st["q"].copy_(torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        st["k"].copy_(torch.randn(T, KVH, D, generator=torch.Generator().manual_seed(seed + 9)).to(torch.bfloat16))
        q, _, _ = [*run("norm", st), None][:3]
        k, v, _ = run("read", st)
        want.append([t.clone() for t in (q, k, v)])
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        q = run("norm", st)[0]
        k, v, _ = run("read", st)
    for seed in (0, 1, 0):
        st["q"].copy_(torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16))
        st["k"].copy_(torch.randn(T, KVH, D, generator=torch.Generator().manual_seed(seed + 9)).to(torch.bfloat16))
        graph.replay()
        for got, expected in zip((q, k, v), want[seed]):
            assert torch.equal(got, expected)
