"""A call that is refused stays refused: every Module keeps the signatures of the calls that passed its checks, so the same bad call
is made twice, and once more behind a good one; and what it keeps does not grow for ever.  On the CPU: the library is a stand-in that records launches, the tensors say that
they are on a GPU."""
import types

import pytest
import torch

import rgd_triton_amd as rgd
from rgd_triton_amd import _hip
from rgd_triton_amd import functional as F_

BF, HF, FP, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64


class OnGpu(torch.Tensor):
    """a CPU tensor that says it is on a GPU, cuda:0 unless told otherwise"""

    is_cuda = True

    def get_device(self):
        return self.__dict__.get("index", 0)


def gpu(*shape, dtype=BF, index=0):
    t = torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)
    t.index = index
    return t


@pytest.fixture
def launches(monkeypatch):
    """names of the entry points that were called, size queries apart"""
    made = []

    def entry(name):
        def call(*a):
            if name.endswith("_workspace") or name.endswith("_bytes") or name == "rgd_attn_seqlen_q_rounded":
                return 0
            made.append(name)
            return 0

        return call

    monkeypatch.setattr(_hip, "lib", lambda: types.SimpleNamespace(**{n: entry(n) for n in _hip._SIGNATURES}))
    monkeypatch.setattr(_hip, "stream_ptr", lambda device: None)
    monkeypatch.setattr(F_, "_current_device", lambda: 0)
    monkeypatch.setattr(F_, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(F_, "_bias_workspaces", lambda *a: (0, 0))
    monkeypatch.setattr(F_, "_decode_workspace", lambda *a: 0)
    return made


# ------------------------------------------------------------------ one module, its good arguments, and changes that are refused


def _append_args():
    return dict(query=gpu(2, 4, 3, 64), key=gpu(2, 2, 3, 64), value=gpu(2, 2, 3, 64), pos_emb=gpu(2, 48, 32, dtype=FP), k_cache=gpu(6, 16, 2, 64),
                v_cache=gpu(6, 16, 2, 64), page_table=gpu(2, 3, dtype=I32), cache_lens=gpu(2, dtype=I32), new_lens=gpu(2, dtype=I32))


APPEND_BAD = {
    "int64 table": dict(page_table=gpu(2, 3, dtype=I64)),
    "int64 lengths": dict(cache_lens=gpu(2, dtype=I64)),
    "int64 new lengths": dict(new_lens=gpu(2, dtype=I64)),
    "three lengths": dict(cache_lens=gpu(3, dtype=I32)),
    "three new lengths": dict(new_lens=gpu(3, dtype=I32)),
    "a table of three rows": dict(page_table=gpu(3, 3, dtype=I32)),
    "lengths with gaps": dict(cache_lens=gpu(4, dtype=I32)[::2]),
    "table columns with gaps": dict(page_table=gpu(2, 6, dtype=I32)[:, ::2]),
    "three key heads": dict(key=gpu(2, 3, 3, 64), value=gpu(2, 3, 3, 64)),
    "fp32 caches": dict(k_cache=gpu(6, 16, 2, 64, dtype=FP), v_cache=gpu(6, 16, 2, 64, dtype=FP)),
    "caches of two sizes": dict(v_cache=gpu(5, 16, 2, 64)),
    "columns in front": dict(k_cache=gpu(6, 16, 64, 2).transpose(2, 3)),
    "another head dim": dict(k_cache=gpu(6, 16, 2, 32), v_cache=gpu(6, 16, 2, 32)),
    "fp32 query": dict(query=gpu(2, 4, 3, 64, dtype=FP)),
    "fewer values": dict(value=gpu(2, 2, 2, 64)),
    "a short rotary table": dict(pos_emb=gpu(2, 47, 32, dtype=FP)),
    "a wide rotary table": dict(pos_emb=gpu(2, 48, 66, dtype=FP)),
    "an odd rotary table": dict(pos_emb=gpu(2, 48, 31, dtype=FP)),
}


def _decode_args():
    return dict(q=gpu(2, 1, 4, 64), k_cache=gpu(6, 16, 2, 64), v_cache=gpu(6, 16, 2, 64), page_table=gpu(2, 3, dtype=I32), seq_lens=gpu(2, dtype=I32))


DECODE_BAD = {
    "int64 table": dict(page_table=gpu(2, 3, dtype=I64)),
    "int64 lengths": dict(seq_lens=gpu(2, dtype=I64)),
    "three lengths": dict(seq_lens=gpu(3, dtype=I32)),
    "a table of three rows": dict(page_table=gpu(3, 3, dtype=I32)),
    "table columns with gaps": dict(page_table=gpu(2, 6, dtype=I32)[:, ::2]),
    "two tokens": dict(q=gpu(2, 2, 4, 64)),
    "no groups": dict(q=gpu(2, 1, 3, 64)),
    "fp32 query": dict(q=gpu(2, 1, 4, 64, dtype=FP)),
    "fp16 query": dict(q=gpu(2, 1, 4, 64, dtype=HF)),
    "another head dim": dict(q=gpu(2, 1, 4, 32)),
    "caches of two sizes": dict(v_cache=gpu(5, 16, 2, 64)),
    "columns in front": dict(v_cache=gpu(6, 16, 64, 2).transpose(2, 3)),
}

OTHERS = {  # operators over whole sequences: (module, good arguments, refused changes)
    "attention": (rgd.FlashAttention, lambda: dict(q=gpu(2, 8, 4, 64), k=gpu(2, 9, 4, 64), v=gpu(2, 9, 4, 64)),
                  {"fewer values": dict(v=gpu(2, 8, 4, 64)), "two types": dict(k=gpu(2, 9, 4, 64, dtype=HF)), "fewer heads": dict(k=gpu(2, 9, 2, 64), v=gpu(2, 9, 2, 64)),
                   "fp32": dict(q=gpu(2, 8, 4, 64, dtype=FP), k=gpu(2, 9, 4, 64, dtype=FP), v=gpu(2, 9, 4, 64, dtype=FP)),
                   "bias of another size": dict(bias=gpu(1, 1, 7, 9))}),
    "l2": (rgd.L2Normalize, lambda: dict(x=gpu(2, 8, 64)), {"two dimensions": dict(x=gpu(2, 8)), "fp64": dict(x=gpu(2, 8, 64, dtype=torch.float64))}),
    "l2 pair": (rgd.FusedL2Normalize2, lambda: dict(x1=gpu(2, 8, 64), x2=gpu(2, 5, 32)),
                {"two types": dict(x2=gpu(2, 5, 32, dtype=HF)), "two batches": dict(x2=gpu(3, 5, 32))}),
    "head norm": (rgd.FusedHeadLayerNorm, lambda: dict(query=gpu(2, 4, 8, 64), key=gpu(2, 4, 9, 64)),
                  {"fewer heads": dict(key=gpu(2, 2, 9, 64)), "wide heads": dict(query=gpu(2, 4, 8, 260), key=gpu(2, 4, 9, 260))}),
    "rope": (rgd.RoPE, lambda: dict(query=gpu(2, 4, 8, 64), key=gpu(2, 4, 9, 64), pos_emb=gpu(2, 10, 32)),
             {"short table": dict(pos_emb=gpu(2, 9, 32)), "fewer heads": dict(key=gpu(2, 2, 9, 64))}),
    "norm and rope": (rgd.FusedLNRoPE, lambda: dict(query=gpu(2, 4, 8, 64), key=gpu(2, 4, 9, 64), pos_emb=gpu(2, 10, 32)),
                      {"short table": dict(pos_emb=gpu(2, 9, 32)), "wide heads": dict(query=gpu(2, 4, 8, 130), key=gpu(2, 4, 9, 130))}),
    "rms": (lambda: rgd.FusedRMSNorm(64, dtype=BF), lambda: dict(x=gpu(2, 8, 64)), {"another width": dict(x=gpu(2, 8, 32)), "fp64": dict(x=gpu(2, 8, 64, dtype=torch.float64))}),
    "rms pair": (lambda: rgd.FusedRMSNorm2((64, 32), dtype=BF), lambda: dict(x1=gpu(2, 8, 64), x2=gpu(2, 5, 32)),
                 {"two types": dict(x2=gpu(2, 5, 32, dtype=HF)), "two batches": dict(x2=gpu(3, 5, 32))}),
}

EVERY = [(rgd.RoPECacheAppend, _append_args, APPEND_BAD), (rgd.FusedLNRoPECacheAppend, _append_args, APPEND_BAD),
         (rgd.PagedDecodeAttention, _decode_args, DECODE_BAD)] + list(OTHERS.values())
NAMES = ["append", "norm and append", "decode"] + list(OTHERS)
REFUSED = [(i, name) for i, (_, _, bad) in enumerate(EVERY) for name in bad]


def _on_gpu(m):
    """the module, its parameters among the tensors that say they are on a GPU"""
    for name, p in list(m.named_parameters()):
        del m._parameters[name]
        setattr(m, name, p.detach().as_subclass(OnGpu))
    return m


@pytest.mark.parametrize("i,name", REFUSED, ids=[f"{NAMES[i]}: {name}" for i, name in REFUSED])
def test_refused_again(launches, i, name):
    make, good, bad = EVERY[i]
    with torch.no_grad():
        m = _on_gpu(make())
        for _ in range(3):
            with pytest.raises((AssertionError, RuntimeError, ValueError)):
                m(**{**good(), **bad[name]})
        assert not launches
        m(**good())
        assert len(launches) == 1
        with pytest.raises((AssertionError, RuntimeError, ValueError)):
            m(**{**good(), **bad[name]})
        m(**good())
        assert len(launches) == 2


@pytest.mark.parametrize("weight,kw", [(gpu(32, 4, dtype=torch.float64), {}), (gpu(32, 4), dict(dtype=torch.float64)), (torch.zeros(32, 4), {}),
                                       (gpu(32, 4), dict(seqlen_q=-1)), (gpu(32, 4), dict(seqlen_k=-2)), (gpu(32, 4, 1), {})])
def test_bias_refused_again(launches, monkeypatch, weight, kw):
    monkeypatch.setattr(F_, "_current_device", lambda: None)  # (what a CPU tensor's device has for an index)
    cache = rgd.RelativePositionBias(32, 4).cache
    call = {**dict(seqlen_q=5, seqlen_k=7, kernel_cache=cache), **kw}
    with torch.no_grad():
        for _ in range(3):
            with pytest.raises((AssertionError, RuntimeError, ValueError)):
                rgd.relative_position_bias_fn(weight, **call)
        assert not launches
        rgd.relative_position_bias_fn(gpu(32, 4), 5, 7, kernel_cache=cache)
        assert len(launches) == 1


MOVED = [(i, name, where) for i, (_, good, _) in enumerate(EVERY) for name in good() for where in (("cpu", "cuda:1") if i < 3 else ("cpu",))]


@pytest.mark.parametrize("i,name,where", MOVED, ids=[f"{NAMES[i]}: {name} on {where}" for i, name, where in MOVED])
def test_each_tensor_on_another_device(launches, i, name, where):
    """behind a good call of the same sizes: a tensor in host memory is refused by every operator, and by those that a serving loop calls
    one on another GPU too"""
    make, good, _ = EVERY[i]
    with torch.no_grad():
        m = _on_gpu(make())
        m(**good())
        assert len(launches) == 1
        t = good()[name]
        other = t.as_subclass(torch.Tensor) if where == "cpu" else gpu(*t.shape, dtype=t.dtype, index=1)
        for _ in range(2):
            with pytest.raises(AssertionError):
                m(**{**good(), name: other})
        assert len(launches) == 1


def test_decode_bias_weight_on_another_device(launches):
    m, good, w = rgd.PagedDecodeAttention(), _decode_args(), gpu(32, 4, dtype=FP)
    rel = lambda w: types.SimpleNamespace(weight=w, max_distance=128, bidirectional=True)  # noqa: E731
    with torch.no_grad():
        m(**good, rel_bias=rel(w))
        for other in (torch.zeros(32, 4), gpu(32, 4, dtype=FP, index=1)):
            with pytest.raises(AssertionError):
                m(**good, rel_bias=rel(other))
    assert len(launches) == 1


def test_signatures_of_a_serving_loop_are_bounded(launches, monkeypatch):
    """queries at other offsets and over other lengths, chunk after chunk, add nothing; prompts of every length stop at a bound"""
    monkeypatch.setattr(F_, "_MOST_SIGNATURES", 64)
    monkeypatch.setattr(F_, "_current_device", lambda: None)
    cache = rgd.RelativePositionBias(32, 4).cache
    w = gpu(32, 4)
    with torch.no_grad():
        for step in range(2 * F_._MOST_SIGNATURES):
            rgd.relative_position_bias_fn(w, 0, step, q_offset=step, kernel_cache=cache)
        assert len(cache.fwd) == 1
        monkeypatch.setattr(F_, "_current_device", lambda: 0)
        m = rgd.RoPECacheAppend()
        for T in range(2 * F_._MOST_SIGNATURES + 7):
            m(**{**_append_args(), **dict(query=gpu(2, 4, T, 64), key=gpu(2, 2, T, 64), value=gpu(2, 2, T, 64))})
            assert len(m.cache.fwd) <= F_._MOST_SIGNATURES
        assert len(m.cache.fwd) == 7
        # still a check for whoever comes behind
        with pytest.raises(AssertionError):
            m(**{**_append_args(), **APPEND_BAD["int64 lengths"]})


# ------------------------------------------------------------------ derivatives that are not there


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(launches, monkeypatch, grad):
    """a tensor that carries a tangent would give a result without one; outside of its level, and beside other levels, calls go on"""
    from torch.autograd import forward_ad

    def dual(t):
        return forward_ad.make_dual(t, torch.ones_like(t))

    monkeypatch.setattr(F_, "_current_device", lambda: None)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        w = gpu(32, 4, dtype=FP)
        with pytest.raises(AssertionError, match="forward-mode"):
            rgd.relative_position_bias_fn(dual(w), 5, 7)
        rgd.relative_position_bias_fn(w, 5, 7)
        monkeypatch.setattr(F_, "_current_device", lambda: 0)
        for name in ("query", "key", "value", "pos_emb", "k_cache", "v_cache"):
            args = _append_args()
            with pytest.raises(AssertionError, match="forward-mode"):
                rgd.RoPECacheAppend()(**{**args, name: dual(args[name])})
        for name in ("q", "k_cache", "v_cache"):
            args = _decode_args()
            with pytest.raises(AssertionError, match="forward-mode"):
                rgd.PagedDecodeAttention()(**{**args, name: dual(args[name])})
        with pytest.raises(AssertionError, match="forward-mode"):
            rgd.paged_decode_attn_func(**_decode_args(), rel_weight=dual(w))
    assert launches == ["rgd_rel_bias_fwd"]
    with torch.no_grad():
        rgd.PagedDecodeAttention()(**_decode_args())
    assert len(launches) == 2


@pytest.mark.gpu
def test_host_memory_behind_a_good_call_on_the_gpu():
    """the same with real tensors: nothing is launched on lengths or tables in host memory"""
    on = lambda args: {n: t.as_subclass(torch.Tensor).cuda() for n, t in args.items()}  # noqa: E731
    with torch.no_grad():
        for m, good, names in ((rgd.RoPECacheAppend(), on(_append_args()), ("page_table", "cache_lens", "new_lens", "pos_emb")),
                               (rgd.PagedDecodeAttention(), on(_decode_args()), ("page_table", "seq_lens", "v_cache"))):
            out = m(**good)
            for name in names:
                for _ in range(2):
                    with pytest.raises(AssertionError):
                        m(**{**good, name: good[name].cpu()})
            assert torch.equal(m(**good), out)


def test_functional_derivatives_are_refused(launches, monkeypatch):
    """torch.func's transforms hand in wrappers without memory of their own"""
    monkeypatch.setattr(F_, "_current_device", lambda: None)
    f = lambda w: rgd.relative_position_bias_fn(w, 5, 7)  # noqa: E731
    w = torch.zeros(32, 4)
    for transform in (lambda: torch.func.jvp(f, (w,), (torch.ones_like(w),)), lambda: torch.func.grad(lambda x: f(x).sum())(w),
                      lambda: torch.func.vmap(f)(torch.zeros(3, 32, 4))):
        with pytest.raises((AssertionError, RuntimeError)):
            transform()
    assert not launches
