"""What the router and the 4-bit products refuse before anything is launched; runs without a GPU."""

import ctypes

import pytest
import torch

from deepep_amd import Router, _lib, ops, w4


@pytest.mark.parametrize("arguments", [
    dict(num_experts=0, num_topk=1), dict(num_experts=1025, num_topk=1), dict(num_experts=8, num_topk=9), dict(num_experts=64, num_topk=33),
    dict(num_experts=8, num_topk=0), dict(num_experts=8, num_topk=2, num_groups=3), dict(num_experts=8, num_topk=2, num_groups=4, num_topk_groups=5),
    dict(num_experts=8, num_topk=5, num_groups=4, num_topk_groups=2), dict(num_experts=8, num_topk=2, score="relu"),
    dict(num_experts=8, num_topk=2, scale=0.0), dict(num_experts=8, num_topk=2, scale=float("nan")), dict(num_experts=8, num_topk=2, scale=float("inf")),
    dict(num_experts=8, num_topk=2, index_dtype=torch.int16), dict(num_experts=8.0, num_topk=2), dict(num_experts=True, num_topk=1),
])
def test_router_arguments(arguments):
    with pytest.raises(ValueError):
        Router(**arguments)


@pytest.mark.parametrize("arguments", [
    dict(num_experts=256, num_topk=2, num_groups=128), dict(num_experts=8, num_topk=2, scale=1e-31), dict(num_experts=8, num_topk=2, scale=-1e31),
    dict(num_experts=8, num_topk=2, scale="1"),
])
def test_router_limits(arguments):
    with pytest.raises(ValueError):
        Router(**arguments)


def test_parameters_are_fixed_and_survive_copies():
    """One set of parameters serves the native and the Python path: it cannot change under either of them."""
    import copy
    import pickle

    class Named(Router):
        pass

    parameters = dict(num_experts=64, num_topk=6, score="sigmoid", normalize=False, scale=2.5, num_groups=8, num_topk_groups=3, index_dtype=torch.int32)
    router = Named(**parameters)
    router.layer = 7
    for name, value in parameters.items():
        assert getattr(router, name) == value
        with pytest.raises(AttributeError):
            setattr(router, name, value)
    for other in (copy.copy(router), copy.deepcopy(router), pickle.loads(pickle.dumps(Router(**parameters)))):
        assert {name: getattr(other, name) for name in parameters} == parameters and isinstance(other, Router)
        assert type(other._native) is type(router._native) and bytes(other._spec()) == bytes(router._spec())
    assert copy.deepcopy(router).layer == 7 and type(copy.copy(router)) is Named


def test_c_abi_limits():
    lib = _lib.load()

    def refused(spec, tokens, word):
        assert lib.dpep_route(ctypes.byref(spec), None, None, None, tokens, None, None, None) == -1
        assert word in lib.dpep_last_error().decode()

    refused(ops.RouterSpec(256, 4, 128, 1, 0, 1, 1.0, 0, 8), 1, "num_groups")
    refused(ops.RouterSpec(16, 4, 1, 1, 0, 1, 1e-31, 0, 8), 1, "scale")
    refused(ops.RouterSpec(16, 4, 1, 1, 0, 1, 1.0, 0, 8), (1 << 30) + 1, "num_tokens")
    big = ops._W4(256, 256, None, (1 << 30) + 1, 128, 32)
    assert lib.dpep_w4_matvec(ctypes.byref(big), 1, 256, 1, 256, None) == -1 and "N=" in lib.dpep_last_error().decode()


def test_routes_of_a_balance_loss_fit_32_bits():
    """A sequence's routes are added up in 32 bits: a batch of 2^31 and more has no loss and no gradient of one.  (Without buffers, so
    that nothing is launched.)"""
    lib = _lib.load()
    spec = ops.RouterSpec(16, 16, 1, 1, 0, 1, 1.0, 0, 8)
    from_weights = ops._RouterGradients(None, None, 256, 256, None, None, None, None, None, 1)
    from_losses = ops._RouterGradients(None, None, 256, 256, None, 256, 256, 256, None, 1)
    calls = (lambda tokens: lib.dpep_balance_loss(ctypes.byref(spec), None, None, tokens, None, 1, 256, 256, 256, 256, None),
             lambda tokens: lib.dpep_route_balance(ctypes.byref(spec), None, None, None, tokens, None, 1, None, None, 256, 256, 256, 256, None),
             lambda tokens: lib.dpep_router_backward(ctypes.byref(spec), ctypes.byref(from_losses), tokens, None))
    for call in calls:
        assert call(1 << 27) == -1 and "T*K" in lib.dpep_last_error().decode()
        assert call((1 << 27) - 1) == -1 and "NULL" in lib.dpep_last_error().decode()
    assert lib.dpep_router_backward(ctypes.byref(spec), ctypes.byref(from_weights), 1 << 27, None) == -1 and "NULL" in lib.dpep_last_error().decode()


def test_c_abi_refuses_before_it_launches():
    lib = _lib.load()
    spec = ops.RouterSpec(16, 4, 1, 1, 0, 1, 1.0, 0, 8)

    def message():
        return lib.dpep_last_error().decode()

    assert lib.dpep_route(None, None, None, None, 1, None, None, None) == -1 and "NULL" in message()
    assert lib.dpep_route(ctypes.byref(spec), None, None, None, 1, None, None, None) == -1 and "NULL" in message()
    assert lib.dpep_route(ctypes.byref(spec), None, None, None, -1, None, None, None) == -1 and "num_tokens" in message()
    assert lib.dpep_route(ctypes.byref(spec), None, None, None, 0, None, None, None) == 0
    assert lib.dpep_route(ctypes.byref(spec), None, ctypes.c_void_p(64), None, 0, None, None, None) == -1 and "bias" in message()
    for field, value, word in (("num_experts", 2000, "num_experts"), ("num_topk", 17, "num_topk"), ("num_groups", 3, "num_groups"), ("num_topk_groups", 2, "num_topk_groups"),
                               ("score", 2, "score"), ("logits_type", 3, "logits_type"), ("index_bytes", 2, "index_bytes"), ("scale", 0.0, "scale")):
        wrong = ops.RouterSpec(16, 4, 1, 1, 0, 1, 1.0, 0, 8)
        setattr(wrong, field, value)
        assert lib.dpep_route(ctypes.byref(wrong), None, None, None, 0, None, None, None) == -1 and word in message(), field
    assert lib.dpep_balance_loss(ctypes.byref(spec), None, None, 0, None, 2, None, None, None, None, None) == -1 and "num_sequences" in message()
    assert lib.dpep_balance_scratch_bytes(0, 4, 1) == 0 and lib.dpep_balance_scratch_bytes(16, 4, 0) == 0 and lib.dpep_balance_scratch_bytes(16, 0, 1) > 0
    assert lib.dpep_router_backward(ctypes.byref(spec), None, 0, None) == -1 and "NULL" in message()
    assert lib.dpep_router_backward(ctypes.byref(spec), ctypes.byref(ops._RouterGradients()), 0, None) == -1 and "neither" in message()


def test_w4_refuses_before_it_launches():
    lib = _lib.load()

    def message():
        return lib.dpep_last_error().decode()

    def matrix(n=64, k=128, group=32, packed=256, scales=256):
        return ctypes.byref(ops._W4(packed, scales, None, n, k, group))

    assert lib.dpep_w4_matvec(None, 1, None, 1, None, None) == -1 and "NULL" in message()
    assert lib.dpep_w4_matvec(matrix(), 0, None, 1, None, None) == -1 and "type" in message()
    assert lib.dpep_w4_matvec(matrix(group=48), 1, None, 1, None, None) == -1 and "group" in message()
    assert lib.dpep_w4_matvec(matrix(group=192, k=384), 1, None, 1, None, None) == -1 and "group" in message()
    assert lib.dpep_w4_matvec(matrix(k=96, group=64), 1, None, 1, None, None) == -1 and "group" in message()
    assert lib.dpep_w4_matvec(matrix(packed=264), 1, None, 1, None, None) == -1 and "aligned" in message()
    assert lib.dpep_w4_matvec(matrix(), 1, None, -1, None, None) == -1 and "num_rows" in message()
    assert lib.dpep_w4_matvec(matrix(), 1, None, 0, None, None) == 0
    assert lib.dpep_w4_matvec(matrix(), 1, None, 1, None, None) == -1 and "NULL" in message()

    def experts(gate_up, down, tokens=4, topk=2, index_bytes=8, local=4):
        return lib.dpep_w4_experts(gate_up, down, 1, None, None, index_bytes, None, tokens, topk, 0, local, None, None, None)

    assert experts(matrix(n=128, k=64), matrix(n=64, k=96)) == -1 and "belong" in message()
    assert experts(matrix(n=128, k=64), matrix(n=64, k=64), tokens=1025) == -1 and "routes" in message()
    assert experts(matrix(n=128, k=64), matrix(n=64, k=64), topk=33) == -1 and "slots" in message()
    assert experts(matrix(n=128, k=64), matrix(n=64, k=64), local=1025) == -1 and "num_local" in message()
    assert experts(matrix(n=128, k=64), matrix(n=64, k=64), index_bytes=2) == -1 and "index_bytes" in message()
    assert experts(matrix(n=128, k=64), matrix(n=64, k=64), tokens=0) == 0
    assert experts(matrix(n=128, k=64), matrix(n=64, k=64)) == -1 and "NULL" in message()
    assert lib.dpep_w4_experts_scratch_bytes(-1, 2, 64, 64) == 0 and lib.dpep_w4_experts_scratch_bytes(4, 2, 64, 64) > 0


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_quantize_rounds_to_half_a_step(symmetric, group):
    gen = torch.Generator().manual_seed(group)
    weight = torch.randn((3, 5, 256), generator=gen)
    held = w4.quantize(weight, group, symmetric=symmetric, dtype=torch.float16)
    assert held.packed.shape == (3, 5, 128) and held.scales.shape == (3, 5, 256 // group) and (held.zeros is None) == symmetric
    step = held.scales.float().repeat_interleave(group, dim=-1)
    # half a step; a zero point that is rounded, and a scale that is (2^-11 of 15 steps), may cut the ends by another half
    assert ((w4.dequantize(held) - weight).abs() <= step * (0.51 if symmetric else 1.02)).all()
    with pytest.raises(ValueError):
        w4.quantize(weight, 48)
    with pytest.raises(ValueError):
        w4.quantize(weight[..., :250], 128)


def test_sizes_are_refused_in_full_and_before_anything_is_allocated(monkeypatch):
    """Sizes that 32 bits do not hold must not come through as what is left of them (2^32 + 5 tokens as 5), and a call beyond a limit
    is refused for its size, not for the memory that its scratch would take.  Tensors without memory stand for those on a GPU."""
    monkeypatch.setattr(ops, "_require", lambda name, t, *rest, **device: t)

    def allocates(*_, **__):
        raise AssertionError("allocated")

    single = {dtype: torch.zeros((), dtype=dtype, device="meta") for dtype in (torch.int64, torch.int32, torch.float32, torch.bfloat16, torch.uint8)}

    def shaped(shape, dtype):
        return single[dtype].expand(shape)

    many = (1 << 32) + 5
    routes, weights = shaped((1 << 27, 16), torch.int64), shaped((1 << 27, 16), torch.float32)
    logits, losses, ids = shaped((1 << 27, 16), torch.bfloat16), shaped((1,), torch.float32), shaped((many, 1), torch.int64)
    router = Router(16, 16)
    balance = (losses, shaped((1, 16), torch.int32), shaped((1,), torch.int32), None)
    from deepep_amd import BalanceLoss

    def matrix(n, k, experts=None):
        lead = () if experts is None else (experts,)
        return w4.W4Weights(shaped((*lead, n, k // 2), torch.uint8), shaped((*lead, n, k // 32), torch.bfloat16))

    def experts(tokens, topk, inter, hidden, local):
        return lambda: w4.expert_ffn(shaped((tokens, hidden), torch.bfloat16), shaped((tokens, topk), torch.int32), shaped((tokens, topk), torch.float32),
                                     matrix(2 * inter, hidden, local), matrix(hidden, inter, local))

    calls = {
        "tokens": [lambda: Router(1, 1).route(shaped((many, 1), torch.bfloat16)), lambda: Router(1, 1).balance_loss(shaped((many, 1), torch.bfloat16), ids),
                   lambda: Router(1, 1).backward(shaped((many, 1), torch.bfloat16), ids, topk_weights=ids, grad_weights=ids)],
        "routes": [lambda: router.route_with_balance(logits), lambda: router.balance_loss(logits, routes),
                   lambda: router.backward(logits, routes, balance=BalanceLoss(*balance), grad_losses=losses),
                   experts(1 << 20, 32, 16384, 32, 1), experts(many, 1, 32, 32, 1)],
        "sequences": [lambda: Router(1, 1).balance_loss(shaped((4, 1), torch.bfloat16), shaped((4, 1), torch.int64), shaped((many,), torch.int32))],
        "N": [lambda: w4.matvec(shaped((1, 32), torch.bfloat16), matrix(many, 32))],
        "K": [lambda: w4.matvec(shaped((1, 1 << 15), torch.bfloat16), matrix(1, 1 << 15))],
        "rows": [lambda: w4.matvec(shaped((many, 32), torch.bfloat16), matrix(1, 32))],
        "topk": [experts(1, many, 32, 32, 1)], "experts": [experts(1, 1, 32, 32, many)],
    }
    monkeypatch.setattr(torch, "empty", allocates)
    monkeypatch.setattr(torch, "empty_like", allocates)
    for what, refused in calls.items():
        for call in refused:
            with pytest.raises(ValueError, match=f"^{what}="):
                call()
    lib = _lib.load()
    assert lib.dpep_balance_scratch_bytes(16, (1 << 30) + 1, 1) == 0 and lib.dpep_balance_scratch_bytes(1025, 4, 1) == 0


@pytest.mark.parametrize("begin", [1.5, "1", None, -1, 1 << 31, (1 << 32) + 1, torch.tensor(0.5)])
def test_first_expert_is_an_integer_of_31_bits(monkeypatch, begin):
    """1.5 must not come through as 1, nor 2^32 + 1."""
    monkeypatch.setattr(ops, "_require", lambda name, t, *rest, **device: t)

    def shaped(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype)

    matrix = w4.W4Weights(shaped(2, 64, 16, dtype=torch.uint8), shaped(2, 64, 1))
    down = w4.W4Weights(shaped(2, 32, 16, dtype=torch.uint8), shaped(2, 32, 1))
    with pytest.raises(ValueError, match="expert_begin"):
        w4.expert_ffn(shaped(1, 32), shaped(1, 1, dtype=torch.int32), shaped(1, 1, dtype=torch.float32), matrix, down, expert_begin=begin)


def test_results_do_not_overlap_what_is_still_read():
    lib = _lib.load()
    matrix = ops._W4(1 << 20, 2 << 20, 3 << 20, 64, 64, 32)
    x, row = 4 << 20, 128
    for y in (x, x + 2, x + 3 * row - 2, x - 3 * row + 2, 1 << 20, (1 << 20) + 64 * 32 - 2, 2 << 20, (2 << 20) + 64 * 4 - 2, (3 << 20) + 64 * 2 - 2):
        assert lib.dpep_w4_matvec(ctypes.byref(matrix), 1, x, 3, y, None) == -1 and "overlap" in lib.dpep_last_error().decode()
    gate_up, down = ops._W4(1 << 20, 2 << 20, None, 64, 32, 32), ops._W4(1 << 20, 2 << 20, None, 32, 32, 32)
    ids = 5 << 20
    for y in (ids, ids + 3 * 2 * 8 - 2, ids - 3 * 64 + 2):
        assert lib.dpep_w4_experts(ctypes.byref(gate_up), ctypes.byref(down), 1, x, ids, 8, 256, 3, 2, 0, 2, y, 6 << 20, None) == -1
        assert "overlap" in lib.dpep_last_error().decode()


@pytest.mark.parametrize("group", [0, -32, -128, 16, 192, 512])
def test_quantize_refuses_groups(group):
    with pytest.raises(ValueError):
        w4.quantize(torch.ones(4, 256), group)


def test_sequences_of_a_launch():
    """A workgroup of 1024 lanes takes a sequence, and a launch holds fewer than 2^32 lanes: more are refused, and not by the launch of
    the second kernel when the first has run.  (Without logits, so that nothing is launched.)"""
    lib = _lib.load()
    spec = ops.RouterSpec(16, 4, 1, 1, 0, 1, 1.0, 0, 8)
    calls = (lambda sequences: lib.dpep_balance_loss(ctypes.byref(spec), None, None, 8, 256, sequences, 256, 256, 256, 256, None),
             lambda sequences: lib.dpep_route_balance(ctypes.byref(spec), None, None, None, 8, 256, sequences, None, None, 256, 256, 256, 256, None))
    for call in calls:
        assert call(1 << 22) == -1 and "num_sequences" in lib.dpep_last_error().decode()
        assert call((1 << 22) - 1) == -1 and "NULL" in lib.dpep_last_error().decode()
