"""CPU-side checks of the operators on learned tables (lookup, its gradient, AdamW): every
argument that a kernel would index with is refused before the device is touched, by the C entry
points as an error string and by the Python functions as an exception."""
import ctypes

import numpy as np
import pytest
import torch

import arboretum_b200 as arb

LIB = arb.lib()
P = ctypes.c_void_p(1 << 20)  # an address that is never followed: the checks come first


def _message(e):
    assert e is not None
    return e.decode()


def _embedding(**change):
    a = dict(table=P, type=0, rows=10, dim=4, row_stride=4, tokens=P, token_bytes=4, bags=3, per_bag=2, bag_stride=2,
             token_stride=1, scale=1.0, out=P, out_type=0, out_stride=4, device=0, stream=None)
    a.update(change)
    return LIB.AEmbedding(*a.values())


@pytest.mark.parametrize("change,words", [
    (dict(token_bytes=2), "int32 or int64"), (dict(bags=-1), "negative"), (dict(per_bag=-1), "negative"),
    (dict(bags=1 << 20, per_bag=1 << 11), "2^31 - 2 tokens"), (dict(bags=1 << 62, per_bag=1 << 62), "2^31 - 2 tokens"),
    (dict(rows=(1 << 31) - 1), "rows"), (dict(rows=-1), "rows"),
    (dict(tokens=None), "tokens is NULL"), (dict(tokens=ctypes.c_void_p((1 << 20) + 2)), "aligned"),
    (dict(table=None), "table is NULL"), (dict(table=ctypes.c_void_p((1 << 20) + 2)), "aligned"),
    (dict(type=3), "element type"), (dict(type=-1), "element type"), (dict(out_type=1), "input's type or fp32"),
    (dict(type=1, out_type=2), "input's type or fp32"), (dict(out=None), "out is NULL"),
    (dict(out_stride=3), "overlap"), (dict(row_stride=-4), "stride"), (dict(row_stride=1 << 45), "stride"),
    (dict(dim=-1), "width"), (dict(token_stride=1 << 60), "stride"),
])
def test_embedding_refuses(change, words):
    assert words in _message(_embedding(**change))


def test_nothing_to_do_touches_no_device():
    assert _embedding(bags=0, tokens=None, out=None) is None
    assert _embedding(dim=0, table=None, out=None) is None


def test_order_and_gradient_refuse():
    a, b = ctypes.c_int64(0), ctypes.c_int64(0)
    for bags, per_bag, rows in ((50, 2, 10), (200000, 1, 10), (200000, 100, 6400)):
        assert LIB.ATokenOrderBytes(bags, per_bag, rows, ctypes.byref(a), ctypes.byref(b)) is None
        assert a.value >= 2 * bags * per_bag + 4 * (rows + 1) and b.value >= 0 and a.value % 256 == 0 and b.value % 256 == 0
    assert "2^31 - 2 tokens" in _message(LIB.ATokenOrderBytes(1 << 30, 2, 10, ctypes.byref(a), ctypes.byref(b)))
    assert "NULL" in _message(LIB.ATokenOrderBytes(1, 1, 10, None, ctypes.byref(b)))
    assert "NULL" in _message(LIB.ATokenOrder(P, 4, 3, 1, 1, 0, 10, None, P, 0, None))
    assert "aligned" in _message(LIB.ATokenOrder(P, 4, 3, 1, 1, 0, 10, ctypes.c_void_p(8), P, 0, None))
    assert "rows" in _message(LIB.ATokenOrder(P, 4, 3, 1, 1, 0, 1 << 31, P, P, 0, None))

    def grad(**change):
        g = dict(grad=P, type=0, bags=3, dim=4, grad_stride=4, order=P, per_bag=1, rows=10, scale=1.0, out=P, out_type=0,
                 out_stride=4, accumulate=0, scratch=P, device=0, stream=None)
        g.update(change)
        return LIB.AEmbeddingGrad(*g.values())
    for change, words in ((dict(order=None), "order is NULL"), (dict(grad=None), "grad is NULL"), (dict(out=None), "out is NULL"),
                          (dict(out_stride=2), "overlap"), (dict(type=2, out_type=1), "input's type"), (dict(rows=-1), "rows"),
                          (dict(per_bag=-1), "negative"), (dict(grad_stride=-1), "stride"), (dict(scratch=ctypes.c_void_p(3)), "aligned"),
                          (dict(bags=1 << 40), "2^31 - 2 tokens")):
        assert words in _message(grad(**change)), change
    assert grad(rows=0, out=None) is None and grad(dim=0, grad=None, out=None) is None


def test_adamw_refuses():
    from arboretum_b200.adamw import _Config, _Param
    params = (_Param * 2)(_Param(1 << 20, 5, 0), _Param(1 << 21, 300, 1))
    n, w = ctypes.c_int64(0), ctypes.c_int64(0)
    assert LIB.AAdamWBytes(params, 2, ctypes.byref(n), ctypes.byref(w)) is None
    assert n.value == 128 + 384 and w.value > 0
    bad = (_Param * 1)(_Param(1 << 20, -5, 0))
    assert "size" in _message(LIB.AAdamWBytes(bad, 1, ctypes.byref(n), ctypes.byref(w)))
    assert "NULL" in _message(LIB.AAdamWBytes(None, 1, ctypes.byref(n), ctypes.byref(w)))
    h = ctypes.c_void_p()

    def create(table=params, count=2, workspace=P, **change):
        c = dict(beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, state_bits=32, seed=0, moment1=1 << 20, moment2=1 << 20,
                 scale1=None, scale2=None, master=None)
        c.update(change)
        return LIB.AAdamWCreate(table, count, ctypes.byref(_Config(*c.values())), workspace, 0, ctypes.byref(h))
    for words, kw in (("state_bits", dict(state_bits=16)), ("betas", dict(beta1=1.0)), ("betas", dict(beta2=-0.1)),
                      ("betas", dict(beta2=float("nan"))), ("eps", dict(eps=float("inf"))), ("eps", dict(weight_decay=-1.0)),
                      ("moment", dict(moment1=None)), ("scale", dict(state_bits=8)), ("aligned", dict(moment2=(1 << 20) + 4)),
                      ("NULL", dict(workspace=None)), ("aligned", dict(workspace=ctypes.c_void_p(16))),
                      ("element type", dict(table=(_Param * 1)(_Param(1 << 20, 5, 7)), count=1)),
                      ("NULL", dict(table=(_Param * 1)(_Param(None, 5, 0)), count=1)),
                      ("aligned", dict(table=(_Param * 1)(_Param((1 << 20) + 2, 5, 0)), count=1))):
        assert words in _message(create(**kw)), kw
    assert "NULL" in _message(LIB.AAdamWStep(None, None, 0, 0, 1e-3, None, None, None))
    assert "NULL" in _message(LIB.AAdamWSetStep(None, 0, None))
    assert LIB.AFreeAdamW(None) is None


def test_python_refusals():
    t = torch.zeros(5, 4)
    i = torch.zeros(3, dtype=torch.int64)
    for error, words, call in (
            (TypeError, "torch tensor", lambda: arb.embedding(i, np.zeros((5, 4), np.float32))),
            (TypeError, "torch tensor", lambda: arb.embedding([1, 2], t)),
            (TypeError, "float32", lambda: arb.embedding(i, t.double())),
            (TypeError, "int32 or int64", lambda: arb.embedding(i.float(), t)),
            (ValueError, "two dimensions", lambda: arb.embedding(i, t[0])),
            (ValueError, "contiguous", lambda: arb.embedding(i, torch.zeros(4, 5).t())),
            (ValueError, "bags x tokens", lambda: arb.embedding(i, t, pooled=True)),
            (ValueError, "requires grad", lambda: arb.embedding(i, t.clone().requires_grad_())),
            (ValueError, "CUDA", lambda: arb.embedding(i, t)),
            (ValueError, "must have shape", lambda: arb.embedding_grad(torch.zeros(4, 4), i, 5)),
            (ValueError, "must have shape", lambda: arb.embedding_grad(torch.zeros(3, 2, 4), i.view(3, 1), 5, pooled=True)),
            (ValueError, "accumulate", lambda: arb.embedding_grad(torch.zeros(3, 4), i, 5, accumulate=True)),
            (arb.ArboretumError, "rows", lambda: arb.embedding_grad(torch.zeros(3, 4), i, 1 << 31)),
            (ValueError, "CUDA", lambda: arb.embedding_grad(torch.zeros(3, 4), i, 5)),
            (arb.ArboretumError, "rows", lambda: arb.token_order(i, -1)),
            (ValueError, "CUDA", lambda: arb.token_order(i, 5)),
            (ValueError, "empty", lambda: arb.AdamW([])),
            (ValueError, "not contiguous", lambda: arb.AdamW([torch.zeros(4, 5).t()])),
            (ValueError, "share memory", lambda: arb.AdamW([t, t[2:]])),
            (ValueError, "state_bits", lambda: arb.AdamW([t], state_bits=4)),
            (TypeError, "float32", lambda: arb.AdamW([i])),
            (TypeError, "lr", lambda: arb.AdamW([t], lr=torch.zeros(2))),
            (ValueError, "CUDA", lambda: arb.AdamW([t]))):
        with pytest.raises(error, match=words):
            call()


def test_leaf_entry_points_refuse():
    import json
    h = ctypes.c_void_p()
    cfg = {"objective": 0, "method": 1, "tree": {"max_depth": 2}}
    assert LIB.AInitGarden(json.dumps(cfg).encode(), ctypes.byref(h)) is None
    n = ctypes.c_int(-1)
    assert LIB.ATreeCount(h, ctypes.byref(n)) is None and n.value == 0
    assert "NULL" in _message(LIB.ATreeCount(None, ctypes.byref(n))) and "NULL" in _message(LIB.ALeafTokens(h, None, -1, P))
    assert "NULL" in _message(LIB.ARefineLeaves(h, None, 1, 0.1, 0.9, 0.99, 1e-8, 0.0, 32))
    data = arb.DMatrix(np.zeros((3, 2), np.float32), y=np.zeros(3, np.float32))
    for words, a in (("negative", (-1, 0.1, 0.9, 0.99, 1e-8, 0.0, 32)), ("state_bits", (1, 0.1, 0.9, 0.99, 1e-8, 0.0, 16)),
                     ("finite", (1, float("nan"), 0.9, 0.99, 1e-8, 0.0, 32)), ("no tree", (1, 0.1, 0.9, 0.99, 1e-8, 0.0, 32))):
        assert words in _message(LIB.ARefineLeaves(h, data.handle, *a))
    assert "n_rounds" in _message(LIB.ALeafTokens(h, data.handle, -2, P))
    assert LIB.ALeafTokens(h, data.handle, -1, P) is None  # no trees: nothing to write
    assert LIB.AFreeGarden(h) is None


@pytest.mark.parametrize("eps,refused", [(1e-40, True), (2.0 ** -127, True), (5e-324, True), (0.0, False), (2.0 ** -126, False)])
def test_adamw_refuses_an_eps_that_the_kernel_takes_for_zero(eps, refused):
    """Below float32's smallest normal number the step would divide zero by zero where no gradient came."""
    from arboretum_b200.adamw import _Config, _Param
    h = ctypes.c_void_p()
    config = _Config(0.9, 0.99, eps, 0.0, 32, 0, 1 << 20, 1 << 20, None, None, None)
    # an address that is no address of the workspace's alignment ends the accepted ones before the device
    e = _message(LIB.AAdamWCreate((_Param * 1)(_Param(1 << 20, 5, 0)), 1, ctypes.byref(config), ctypes.c_void_p(16), 0, ctypes.byref(h)))
    assert ("2^-126" in e) == refused and ("aligned" in e) != refused


@pytest.mark.parametrize("scale", [float("inf"), -float("inf"), float("nan"), 1e39])
def test_scale_is_finite(scale):
    """Zeros of empty bags and unnamed rows would become NaN."""
    assert "scale" in _message(_embedding(scale=scale))
    assert "scale" in _message(LIB.AEmbeddingGrad(P, 0, 3, 4, 4, P, 1, 10, scale, P, 0, 4, 0, P, 0, None))


def test_tensors_whose_memory_is_gone_are_refused():
    """A storage can be freed or shrunk under its tensors; a view's address is then that of nothing."""
    t = torch.zeros(5, 4)
    i = torch.zeros(3, dtype=torch.int64)
    for size in (0, 4 * 15):
        base = torch.zeros(24)
        view, last = base[4:].view(5, 4), base[12:].view(3, 4)
        base.untyped_storage().resize_(size)
        for call in (lambda: arb.embedding(i, view), lambda: arb.embedding_grad(last, i, 5)):
            with pytest.raises(ValueError, match="memory"):
                call()
    gone = torch.zeros(4, dtype=torch.int64)[1:]
    gone.untyped_storage().resize_(0)
    for call in (lambda: arb.embedding(gone, t), lambda: arb.token_order(gone, 5), lambda: arb.embedding_grad(torch.zeros(3, 4), gone, 5)):
        with pytest.raises(ValueError, match="memory"):
            call()
    with pytest.raises(ValueError, match="memory"):
        arb.embedding(i, t.to_sparse())


def test_tensors_with_tangents_are_refused():
    """Forward-mode derivatives are not followed, so they are not dropped either."""
    from torch.autograd import forward_ad
    i = torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        table = forward_ad.make_dual(torch.zeros(5, 4), torch.ones(5, 4))
        grad = forward_ad.make_dual(torch.zeros(3, 4), torch.ones(3, 4))
        for call in (lambda: arb.embedding(i, table), lambda: arb.embedding_grad(grad, i, 5)):
            with pytest.raises(ValueError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="CUDA"):
            arb.embedding(i, forward_ad.unpack_dual(table).primal)
    for call in (lambda t: arb.embedding(i, t), lambda t: arb.embedding_grad(t[:3], i, 5)):
        with pytest.raises(Exception):  # never a result
            torch.func.jvp(call, (torch.zeros(5, 4),), (torch.ones(5, 4),))
        with pytest.raises(Exception):
            torch.vmap(call)(torch.zeros(2, 5, 4))


@pytest.mark.filterwarnings("ignore")
def test_tracing_is_refused():
    """A trace that does not see a call would keep its result as a constant, or unfilled memory."""
    from torch.fx.experimental.proxy_tensor import make_fx
    i = torch.zeros(3, dtype=torch.int64)
    t = torch.zeros(5, 4)
    for call in (lambda x: arb.embedding(i, x), lambda x: arb.embedding_grad(x[:3], i, 5), lambda x: arb.token_order(x[:, 0].long(), 5).rows * x):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (t,))
        with pytest.raises(ValueError, match="traced"):
            make_fx(call)(t)
        with pytest.raises(ValueError, match="CUDA"):
            call(t)


def test_views_to_be_negated_are_refused():
    """The imaginary part of a conjugate is such a view: its memory holds the opposite."""
    i = torch.zeros(3, dtype=torch.int64)
    t = torch.zeros(5, 4)
    part = torch.zeros(5, 1, dtype=torch.complex64).conj().imag
    assert part.is_neg()
    for call in (lambda: arb.embedding(i, part), lambda: arb.embedding(i, torch._neg_view(t)), lambda: arb.embedding_grad(torch._neg_view(t[:3]), i, 5),
                 lambda: arb.embedding_grad(part[:3], i, 5), lambda: arb.embedding(torch._neg_view(i), t), lambda: arb.token_order(torch._neg_view(i), 5)):
        with pytest.raises(ValueError, match="negated"):
            call()
    with pytest.raises(ValueError, match="CUDA"):
        arb.embedding(i, part.resolve_neg())


def test_leaf_tokens_refuse_another_device(monkeypatch):
    """The model's kernel does not write to the memory of a device it does not work on."""
    data = arb.DMatrix(np.zeros((3, 2), np.float32), y=np.zeros(3, np.float32))
    model = arb.Garden({"objective": 0, "method": 1, "tree": {"max_depth": 2}}, data)

    class Out:  # looks like a tensor of the second device, of no trees
        dtype, shape, device = torch.int32, (0, 3), torch.device("cuda", 1)
        is_contiguous = is_inference = lambda self: True
        data_ptr = lambda self: 1 << 20  # noqa: E731
        t = lambda self: self  # noqa: E731

    class Stream:
        synchronize = lambda self: None  # noqa: E731
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: Stream())
    monkeypatch.setattr(arb.Garden, "_device", lambda self: 0, raising=False)
    with pytest.raises(ValueError, match="cuda:1, the model works on cuda:0"):
        model.leaf_tokens(data, out=Out())
    monkeypatch.setattr(arb.Garden, "_device", lambda self: 1, raising=False)
    assert isinstance(model.leaf_tokens(data, out=Out()), Out)
    assert "NULL" in _message(LIB.AModelDevice(None, ctypes.byref(ctypes.c_int(0)))) and "NULL" in _message(LIB.AModelDevice(model.handle, None))


def test_refinement_refuses_a_regression_of_several_outputs():
    """Its loss has one output: the trees of the others would move along a gradient that is none."""
    import json
    cfg = {"objective": 0, "method": 1, "tree": {"max_depth": 1, "labels_count": 2}}
    nodes = [{"id": 0, "leaf": False, "left": 1, "right": 2, "threshold": 0.5, "fid": 0}, {"id": 1, "leaf": True, "idx": 0}, {"id": 2, "leaf": True, "idx": 1}]
    model = arb.Garden(cfg)
    model.load(json.dumps({"configuration": cfg, "model": [{"depth": 2, "nodes": nodes, "weights": [0.25, -0.25]}] * 2}))
    before = model.dump()
    with pytest.raises(arb.ArboretumError, match="labels_count"):
        model.refine_leaves(arb.DMatrix(np.zeros((3, 2), np.float32), y=np.ones(3, np.float32)), 1)
    assert model.dump() == before


@pytest.mark.parametrize("stride", [-2 ** 63, 2 ** 63 - 1, -2 ** 46 - 1, 2 ** 46 + 1])
def test_token_strides_are_bounded_both_ways(stride):
    assert "stride" in _message(_embedding(bag_stride=stride)) and "stride" in _message(_embedding(token_stride=stride))
    for strides in ((stride, 1), (1, stride)):
        assert "stride" in _message(LIB.ATokenOrder(P, 4, 3, 2, strides[0], strides[1], 10, P, P, 0, None))


def test_a_flag_without_a_truth_value():
    """Its own error comes out, not a result with an error behind it."""
    i, t, both = torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4), np.ones(2)
    for call in (lambda: arb.embedding(i, t, pooled=both), lambda: arb.embedding_grad(t, i, 5, pooled=both), lambda: arb.embedding_grad(t, i, 5, out=t, accumulate=both)):
        with pytest.raises(ValueError, match="ambiguous"):
            call()
    with pytest.raises(ValueError, match="ambiguous"):
        arb.lookup._tensors.token_order(i, 5, both)
