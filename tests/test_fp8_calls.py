"""The compiled binding's 8-bit, rotary and page calls (csrc/fp4_calls.cpp) against the wrappers' own checks, as
tests/test_fp4_calls.py: a call that the binding takes does what the wrapper would have done; the rest is left to the
wrapper untouched, so errors are the wrapper's."""

import pytest
import torch

from nano_vllm_ascend_b200 import _calls, ops, ops_fp8

D, H, KVH, BS, NB, T = 128, 8, 2, 32, 6, 5
TAKEN = {"append": (ops_fp8, "_append8"), "read": (ops_fp8, "_read8"), "decode": (ops_fp8, "_decode8"),
         "prefill": (ops_fp8, "_prefill8"), "rotary": (ops, "_rotary"), "copy": (ops, "_copy_blocks"),
         "remap": (ops, "_remap_blocks")}


def state(dev, many=0):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)
    i = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device=dev)
    st = dict(pool=torch.zeros(ops_fp8.pool_shape(NB, BS, KVH), dtype=torch.uint8, device=dev), q=r(T, H, D),
              k=r(T, KVH, D), v=r(T, KVH, D), slots=i([3, 40, 170, 0, 99], torch.int64), wq=r(D), wk=r(D),
              inv=torch.rand(D // 2, generator=g, dtype=torch.float64).to(dev), pos=i([1, 5, 63, 0, 7], torch.int64),
              table=i([[5, 1], [0, 3], [2, 4], [1, 0], [3, 5]]), lens=i([64, 33, 1, 0, 40]), cu=i([0, 1, 2, 3, 4, 5]),
              err=i([0]), scale=0.1, max_q=1, pairs=i([[0, 4], [-1, 2], [3, -1]]), map=i([3, 1, 2, 0, 5, 4]),
              pools=[torch.randint(0, 255, (3, NB, 4, 64), generator=g, dtype=torch.uint8).to(dev) for _ in range(2)],
              interleaved=False, factor=1.5, eps=1e-6, qo=None, ko=None)
    st["out"] = torch.zeros_like(st["q"])
    st["ws"] = torch.zeros(1 << 22, dtype=torch.uint8, device=dev)
    return st


def run(op, st):
    if op == "append":
        ops_fp8.kv_append_fp8(st["pool"], st["k"], st["v"], st["slots"], st["err"])
        return [st["pool"], st["err"]]
    if op == "read":
        return [*ops_fp8.kv_read_fp8(st["pool"], st["slots"], st.get("dtype", torch.bfloat16), error_word=st["err"]),
                st["err"]]
    if op == "decode":
        out = ops_fp8.paged_decode_fp8(st["out"], st["q"], st["pool"], st["table"], st["lens"], st["scale"], st["ws"],
                                       st.get("ctas", 0))
        assert out is st["out"]
        return [out, st["ws"][:4]]
    if op == "prefill":
        out = ops_fp8.paged_prefill_fp8(st["out"], st["q"], st["pool"], st["table"], st["cu"], st["lens"], st["max_q"],
                                        st["scale"], st["err"])
        assert out is st["out"]
        return [out, st["err"]]
    if op == "rotary":
        q, k = ops.rotary(st["q"], st["k"], st["inv"], st["pos"], st["interleaved"], st["factor"], st["wq"], st["wk"],
                          st["eps"], st["qo"], st["ko"])
        assert (st["qo"] is None or q is st["qo"]) and (st["ko"] is None or k is st["ko"])
        return [q, k]
    if op == "copy":
        ops.copy_blocks(st["pools"], st["pairs"], st["err"])
        return [*([st["pools"]] if isinstance(st["pools"], torch.Tensor) else st["pools"]), st["err"]]
    ops.remap_blocks(st["table"], st["map"], st["err"])
    return [st["table"], st["err"]]


def long_append(dev):
    g = torch.Generator().manual_seed(5)
    n = 700
    return dict(pool=torch.zeros(ops_fp8.pool_shape(30, BS, KVH), dtype=torch.uint8, device=dev),
                slots=torch.randperm(30 * BS, generator=g)[:n].to(dev),
                **{x: torch.randn(n, KVH, D, generator=g).to(torch.float16).to(dev) for x in "kv"})


@pytest.mark.gpu
@pytest.mark.parametrize("op,change", [
    ("append", {}), ("append", dict(err=None)), ("append", dict(slots=[3, 192, -1, 0, 9])), ("append", long_append),
    ("read", {}), ("read", dict(dtype=torch.float16)), ("read", dict(slots=[3, 192, -1, 0, 0])),
    ("decode", {}), ("decode", dict(ctas=3)), ("decode", dict(lens=[64, 65, 1, 0, 40])),
    ("prefill", {}), ("prefill", dict(lens=[64, 65, 1, 0, 40])), ("rotary", {}), ("rotary", dict(wq=None, wk=None)),
    ("rotary", dict(interleaved=True)),
    ("rotary", lambda dev: dict(qo=torch.zeros(T, H, D, dtype=torch.bfloat16, device=dev))),
    ("rotary", lambda dev: dict(inv=torch.rand(5, dtype=torch.float64, generator=torch.Generator().manual_seed(2)).to(dev))),
    ("copy", {}), ("copy", dict(pairs=[[0, 6], [-2, 1], [1, 2]])),
    ("copy", lambda dev: dict(pools=torch.arange(2 * NB * 16, device=dev).view(2, NB, 16))),
    ("remap", {}), ("remap", dict(map=[3, 1, 2, 0, 6, 4])), ("remap", dict(map=[1, 0]))])
def test_a_call_that_is_taken_does_what_the_wrapper_does(cuda_device, monkeypatch, op, change):
    assert _calls.binding() is not None, "the binding is built with the library"
    results = []
    for taken in (True, False):
        st = state(cuda_device)
        g = torch.Generator().manual_seed(3)
        every = dict(st, slots=torch.arange(NB * BS, device=cuda_device))
        every.update({x: torch.randn(NB * BS, KVH, D, generator=g).to(torch.bfloat16).to(cuda_device) for x in "kv"})
        run("append", every)
        run("rotary", st), run("copy", dict(st, pairs=st["pairs"][:0]))  # each wrapper's first call loads the binding
        for key, value in (change(cuda_device) if callable(change) else change).items():
            if isinstance(value, list):
                value = torch.tensor(value, dtype=st[key].dtype, device=cuda_device)
            st[key] = value
        seen = []
        module, name = TAKEN[op]
        with monkeypatch.context() as m:
            if taken:
                fast = getattr(_calls.binding(), name[1:])
                m.setattr(module, name, lambda *a: seen.append(fast(*a)) or seen[-1])
            else:
                m.setattr(module, name, _calls._leave)
            results.append([t.clone() for t in run(op, st) if t is not None])
        assert not taken or (seen and not (seen[0].__class__ is int and seen[0] == _calls.NOT_TAKEN))
    for a, b in zip(*results):
        assert a.dtype == b.dtype and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def bad(dev):
    """(operator, what a caller gives wrong): what only the binding could let through."""
    f = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=dev)
    i32, i64, u8, f32, f64 = torch.int32, torch.int64, torch.uint8, torch.float32, torch.float64
    yield "append", dict(k=f(T, KVH, D, t=f32))
    yield "append", dict(k=f(T, KVH, D), v=f(T, KVH, D, t=torch.float16))
    yield "append", dict(k=f(T, KVH, 64), v=f(T, KVH, 64))
    yield "append", dict(k=f(T, KVH + 1, D), v=f(T, KVH + 1, D))
    yield "append", dict(v=f(T + 1, KVH, D))
    yield "append", dict(slots=f(T, t=i32))
    yield "append", dict(slots=f(T + 1, t=i64))
    yield "append", dict(k=f(KVH, T, D).transpose(0, 1), v=f(KVH, T, D).transpose(0, 1))
    yield "append", dict(err=f(1, t=i64))
    yield "append", dict(err=f(0, t=i32))
    yield "append", dict(pool=f(NB, KVH, BS // 16, 4127, t=u8))
    yield "append", dict(pool=f(NB, BS // 16, KVH, 4128, t=u8).transpose(1, 2))
    yield "append", dict(pool=f(NB, KVH, 3, 4128, t=u8))
    yield "append", dict(k=torch.zeros(T, KVH, D, dtype=torch.bfloat16))
    yield "read", dict(slots=f(T, t=i32))
    yield "read", dict(pool=f(NB, KVH, BS // 16, 4128, t=torch.int8))
    yield "read", dict(dtype=f32)
    yield "decode", dict(out=f(T, H, D, t=f32))
    yield "decode", dict(q=f(T, H, 2 * D)[:, :, ::2])
    yield "decode", dict(table=f(T, 2, t=i64))
    yield "decode", dict(table=f(2, T, t=i32).t())
    yield "decode", dict(table=f(1, 2, t=i32).expand(T, 2))
    yield "decode", dict(lens=f(T + 1, t=i32))
    yield "decode", dict(lens=f(2 * T, t=i32)[::2])
    yield "decode", dict(table=f(T + 1, 2, t=i32), lens=f(T + 1, t=i32))
    yield "decode", dict(ws=f(64, t=u8))
    yield "decode", dict(scale=0.0)
    yield "decode", dict(scale=float("nan"))
    yield "decode", dict(ctas=-1)
    yield "decode", dict(q=f(T, 18, D), out=f(T, 18, D))
    yield "prefill", dict(cu=f(T, t=i32))
    yield "prefill", dict(cu=f(T + 1, t=i64))
    yield "prefill", dict(max_q=-1)
    yield "prefill", dict(scale=-1.0)
    yield "prefill", dict(q=f(T, 7, D), out=f(T, 7, D))
    yield "rotary", dict(q=f(T, H, D, t=f32), k=f(T, KVH, D, t=f32))
    yield "rotary", dict(k=f(T, KVH, D, t=torch.float16))
    yield "rotary", dict(k=f(T + 1, KVH, D))
    yield "rotary", dict(k=f(T, KVH, 64))
    yield "rotary", dict(q=f(H, T, D).transpose(0, 1))
    yield "rotary", dict(q=f(1, H, D).expand(T, H, D))
    yield "rotary", dict(inv=f(64, t=f32))
    yield "rotary", dict(inv=f(65, t=f64))
    yield "rotary", dict(inv=f(0, t=f64))
    yield "rotary", dict(inv=f(8, 8, t=f64))
    yield "rotary", dict(pos=f(T, t=i32))
    yield "rotary", dict(pos=f(T - 1, t=i64))
    yield "rotary", dict(wk=None)
    yield "rotary", dict(wq=f(D, t=f32))
    yield "rotary", dict(wk=f(64))
    yield "rotary", dict(qo=f(T, H, D, t=torch.float16))
    yield "rotary", dict(ko=f(T, H, D))
    yield "rotary", dict(pos=torch.zeros(T, dtype=i64))
    yield "copy", dict(pairs=f(3, 2, t=i64))
    yield "copy", dict(pairs=f(6, t=i32))
    yield "copy", dict(pairs=torch.zeros(3, 2, dtype=i32))
    yield "copy", dict(pools=[f(3, NB, 64, t=u8), f(3, NB + 1, 64, t=u8)])
    yield "copy", dict(pools=[f(3, NB, 64, t=u8), f(3, NB, 64, t=torch.int8)])
    yield "copy", dict(pools=f(3, NB, 64, t=u8).transpose(0, 1))
    yield "copy", dict(pools=f(3, NB, 40, t=u8))
    yield "copy", dict(pools=f(3, NB, t=u8))
    yield "copy", dict(err=f(1, t=f32))
    yield "remap", dict(table=f(5, 2, t=i64))
    yield "remap", dict(table=f(2, 5, t=i32).t())
    yield "remap", dict(map=f(6, t=i64))
    yield "remap", dict(map=f(0, t=i32))
    yield "remap", dict(map=f(2, 3, t=i32))
    yield "remap", dict(err=f(0, t=i32))


@pytest.mark.gpu
def test_what_is_wrong_is_refused_as_by_the_wrapper(cuda_device, monkeypatch):
    for op, change in bad(cuda_device):
        messages = []
        for taken in (True, False):
            st = dict(state(cuda_device), **change)
            whole = {n: [t.clone() for t in (st[n] if isinstance(st[n], list) else [st[n]])]
                     for n in ("pool", "out", "pools", "table")}
            with monkeypatch.context() as m:
                if not taken:
                    m.setattr(*TAKEN[op], _calls._leave)
                with pytest.raises((ValueError, RuntimeError)) as e:
                    run(op, st)
            messages.append((e.type, str(e.value)))
            for n, was in whole.items():
                assert all(torch.equal(a, b) for a, b in zip(was, st[n] if isinstance(st[n], list) else [st[n]])), (op, n)
        assert messages[0] == messages[1], (op, list(change))


@pytest.mark.gpu
def test_repairable_arguments_are_repaired(cuda_device):
    """Index tensors, pairs and maps that are strided are copied by the wrapper; numbers may be numpy's."""
    import numpy as np

    for op, names in (("append", ["slots"]), ("read", ["slots"]), ("rotary", ["pos", "inv", "wq"]), ("copy", ["pairs"]),
                      ("remap", ["map"])):
        st, again = state(cuda_device), state(cuda_device)
        want = [t.clone() for t in run(op, st)]
        for name in names:
            t = again[name]
            wide = torch.zeros(2 * t.shape[0], *t.shape[1:], dtype=t.dtype, device=cuda_device)
            wide[::2] = t
            again[name] = wide[::2]
        again["eps"], again["factor"] = np.float64(again["eps"]), np.float32(again["factor"])
        for a, b in zip(run(op, again), want):
            assert torch.equal(a, b), op


def test_host_tensors_are_left_to_the_wrapper():
    c = _calls.binding()
    if c is None:
        pytest.skip("the binding is not built")
    st = state("cpu")
    assert c.append8(st["pool"], st["k"], st["v"], st["slots"], None) == _calls.NOT_TAKEN
    assert c.append8(None, 1, "x", st["slots"], None) == _calls.NOT_TAKEN
    assert c.read8(st["pool"], st["slots"], False, None) == _calls.NOT_TAKEN
    assert c.rotary(st["q"], st["k"], st["inv"], st["pos"], False, 1.0, None, None, 1e-6, None, None) == _calls.NOT_TAKEN
    assert c.copy_blocks(st["pools"][0], st["pools"][1], st["pairs"], None) == _calls.NOT_TAKEN
    assert c.remap_blocks(st["table"], st["map"], None) == _calls.NOT_TAKEN
    with pytest.raises(TypeError, match="3 arguments"):
        c.append8(1, 2, 3)
    for op in TAKEN:
        with pytest.raises(ValueError, match="CUDA|workspace|device|on cpu"):
            run(op, st)


@pytest.mark.gpu
def test_captured_calls_allocate_in_the_graph(cuda_device):
    """What a captured call allocates (outputs, a long append's workspace) belongs to the graph; a replay on new inputs
    writes it again."""
    st = dict(state(cuda_device), **long_append(cuda_device), err=None)
    n = st["slots"].numel()
    st["q"] = torch.zeros(n, H, D, dtype=torch.float16, device=cuda_device)
    st.update(wq=None, wk=None, pos=torch.arange(n, device=cuda_device))

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        for x in "qkv":
            st[x].copy_(torch.randn(st[x].shape, generator=g))
        st["slots"].copy_(torch.randperm(30 * BS, generator=g)[:n])

    def chain():
        q, k = run("rotary", st)
        ops_fp8.kv_append_fp8(st["pool"], k, st["v"], st["slots"])
        return [q, k, *ops_fp8.kv_read_fp8(st["pool"], st["slots"])]

    want = []
    for seed in (0, 1):
        fill(seed)
        st["pool"].zero_()
        want.append([t.clone() for t in chain()])
    stream = torch.cuda.Stream(cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = chain()
    for seed in (0, 1, 0):
        fill(seed)
        st["pool"].zero_()
        graph.replay()
        for a, b in zip(got, want[seed]):
            assert torch.equal(a, b)
