"""lora_linear against its definition in 64 bits (oracle/lora.py), element by element within the bound carried there
(every rounding half a step, every fp32 sum of n products n 2^-24 of its magnitudes) and the result's own rounding."""

import math

import pytest
import torch

from oracle.lora import lora_reference

pytestmark = pytest.mark.gpu


def make(num_tokens, d_model, width, rank, num_adapters, order="requests", seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(num_tokens, d_model, generator=g).bfloat16()
    w = (torch.randn(d_model, width, generator=g) / d_model**0.5).bfloat16()
    a = (torch.randn(num_adapters, rank, d_model, generator=g) / d_model**0.5).bfloat16()
    b = (torch.randn(num_adapters, rank, width, generator=g) / rank**0.5).bfloat16()
    scale = torch.rand(num_adapters, generator=g) + 0.5
    idx = torch.randint(-1, num_adapters, (num_tokens,), generator=g)
    if order == "requests":  # runs of one adapter
        idx = idx.sort().values[torch.arange(num_tokens)] if num_tokens else idx
    elif order == "none":
        idx[:] = -1
    elif order == "one":
        idx[:] = num_adapters - 1
    return [t.cuda() for t in (x, w, a, b, idx, scale)]


def check(x, w, a, b, idx, scale, fp32=False):
    from sparsebench_b200 import lora_linear

    out = lora_linear(x, w, a, b, idx, scale=scale, out_dtype=torch.float32 if fp32 else None)
    assert out.dtype == (torch.float32 if fp32 else torch.bfloat16) and out.shape == (x.shape[0], w.shape[1])
    want, bound = lora_reference(x, w, a, b, idx, scale, fp32)
    half = 2.0**-24 if fp32 else 2.0**-8
    err = (out.double() - want).abs()
    allowed = 1.01 * (bound + half * (want.abs() + bound)) + 2.0**-133
    assert torch.isfinite(out).all()
    assert bool((err <= allowed).all()), f"{float((err / allowed).max()):.3g} times the bound"
    return out


SHAPES = [
    (1, 64, 64, 8, 1), (1, 8, 8, 8, 3), (1, 256, 256, 16, 8), (2, 128, 264, 24, 2), (7, 136, 40, 16, 4), (16, 512, 512, 16, 16),
    (33, 320, 1000, 32, 5), (63, 72, 136, 8, 40), (64, 1024, 256, 64, 9), (65, 256, 128, 16, 3), (127, 200, 520, 40, 6),
    (128, 64, 256, 128, 7), (129, 128, 8, 8, 12), (300, 392, 264, 24, 10), (513, 512, 768, 64, 33), (1000, 264, 88, 48, 4),
    (2049, 128, 64, 8, 16), (4096, 1024, 64, 8, 16),
]


@pytest.mark.parametrize("fp32", [False, True], ids=["bf16", "fp32"])
@pytest.mark.parametrize("order", ["requests", "any"])
@pytest.mark.parametrize(("num_tokens", "d_model", "width", "rank", "num_adapters"), SHAPES)
def test_matches_definition(num_tokens, d_model, width, rank, num_adapters, order, fp32):
    check(*make(num_tokens, d_model, width, rank, num_adapters, order, seed=num_tokens), fp32=fp32)


@pytest.mark.parametrize("num_tokens", [1, 40, 200])
@pytest.mark.parametrize("order", ["none", "one"])
def test_no_adapter_and_one_for_all(num_tokens, order):
    x, w, a, b, idx, scale = make(num_tokens, 256, 320, 16, 4, order)
    out = check(x, w, a, b, idx, scale)
    if order == "none":
        idx[::2] = 4  # past the end: no adapter either
        idx[1::2] = -7
        assert torch.equal(check(x, w, a, b, idx.int(), None), out)


@pytest.mark.parametrize("num_tokens", [1, 40, 200])
def test_ids_that_differ_in_their_upper_half_only(num_tokens):
    x, w, a, b, idx, scale = make(num_tokens, 128, 136, 16, 4, "any")
    idx[::3] = 2**32 + 1
    idx[1::7] = -(2**32) + 2
    out = check(x, w, a, b, idx, scale)
    assert torch.equal(out, check(x, w, a, b, torch.where((idx < 0) | (idx >= 4), -1, idx), scale))


@pytest.mark.parametrize("fp32", [False, True], ids=["bf16", "fp32"])
@pytest.mark.parametrize("width", [648, 2568, 5128])
def test_columns_of_a_tile(width, fp32):
    # Two row tiles: few columns have tiles of 64, more have 128, then 256. One adapter's B is not finite in two columns.
    from sparsebench_b200 import lora_linear

    x, w, a, b, idx, scale = make(130, 72, width, 16, 20, "any", seed=width)
    want = check(x, w, a, b, idx, scale, fp32)
    idx[:3] = 4
    b[4, 2, width - 1] = math.inf
    b[4, 0, 70] = math.nan
    got = lora_linear(x, w, a, b, idx, scale, torch.float32 if fp32 else torch.bfloat16)
    others = idx != 4
    assert torch.equal(got[others], want[others])
    bad = torch.zeros(width, dtype=torch.bool, device="cuda")
    bad[[70, width - 1]] = True
    assert torch.equal(torch.isfinite(got), others[:, None] | ~bad)


@pytest.mark.parametrize("num_tokens", [5, 300])
def test_more_adapters_in_a_tile_than_one_product_holds(num_tokens):
    # 128 tokens of 128 different adapters of rank 128: 64 groups of two adapters each.
    x, w, a, b, idx, scale = make(num_tokens, 128, 72, 128, 140)
    idx = (torch.arange(num_tokens, device="cuda") * 11) % 140
    check(x, w, a, b, idx, scale)
    check(x, w, a, b, idx, scale, fp32=True)


@pytest.mark.parametrize("fp32", [False, True], ids=["bf16", "fp32"])
@pytest.mark.parametrize("num_tokens", [3, 50, 260])
@pytest.mark.parametrize("where", ["a", "b", "x", "scale"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_finite_stays_with_its_request(num_tokens, where, bad, fp32):
    from sparsebench_b200 import lora_linear

    x, w, a, b, idx, scale = make(num_tokens, 192, 328, 16, 5, "any", seed=2)
    idx[0] = 3
    dtype = torch.float32 if fp32 else torch.bfloat16
    want = lora_linear(x, w, a, b, idx, scale, dtype)
    if where == "a":
        a[3, 5, 7] = bad
    elif where == "b":
        b[3, 5, 7] = bad
    elif where == "x":
        x[0, 9] = bad
    else:
        scale[3] = bad
    got = lora_linear(x, w, a, b, idx, scale, dtype)
    theirs = idx == 3
    if where == "x":
        theirs = torch.arange(num_tokens, device="cuda") == 0
    assert torch.equal(got[~theirs], want[~theirs])
    if where == "b":  # one column of the adapter: the others as before, within what another order of the sum changes
        others = torch.arange(328, device="cuda") != 7
        assert not torch.isfinite(got[theirs][:, 7]).any()
        half = 2.0**-24 if fp32 else 2.0**-8
        value, bound = lora_reference(x, w, a, torch.where(torch.isfinite(b), b, torch.zeros_like(b)), idx, scale, fp32)
        err = (got.double() - value).abs()[theirs][:, others]
        assert bool((err <= 1.01 * (bound + half * (value.abs() + bound))[theirs][:, others]).all())
    else:
        assert not torch.isfinite(got[theirs]).any()


@pytest.mark.parametrize("fp32", [False, True], ids=["bf16", "fp32"])
@pytest.mark.parametrize("num_tokens", [3, 50, 260])
def test_infinities_of_an_adapter_come_out_as_the_definition_has_them(num_tokens, fp32):
    # An infinite number of B makes the adapter's rows infinite with the sign of x A^T there, whatever the batch size; two
    # of them with opposite terms, and a NaN, make them NaN. x A^T of these rows is far enough from 0 to have its sign.
    from sparsebench_b200 import lora_linear

    x, w, a, b, idx, scale = make(num_tokens, 192, 328, 16, 5, "any", seed=2)
    idx[0] = 3
    rows = idx == 3
    v = x[rows].double() @ a[3].double().T
    v_abs = x[rows].double().abs() @ a[3].double().abs().T
    b[3, 5, 7] = math.inf
    b[3, 6, 70] = -math.inf
    b[3, 5, 200], b[3, 9, 200] = math.inf, -math.inf
    b[3, 2, 327] = math.nan
    assert bool((v.abs() > 4 * 192 * 2.0**-24 * v_abs)[:, [2, 5, 6, 9]].all())
    value, _ = lora_reference(x, w, a, b, idx, scale, fp32)
    got = lora_linear(x, w, a, b, idx, scale, torch.float32 if fp32 else torch.bfloat16)
    assert int(torch.isinf(value).sum()) >= 2 * int(rows.sum())
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(value)), kind.__name__


def test_rows_behind_the_batch_stay_as_they_were():
    import ctypes

    from sparsebench_b200 import _C, _lib

    lib = _lib.load()
    for num_tokens, width in ((5, 72), (130, 264)):
        x, w, a, b, idx, scale = make(num_tokens, 128, width, 8, 3)
        for fp32, dtype in ((0, torch.bfloat16), (1, torch.float32)):
            room = torch.full((num_tokens + 140, width), 7.0, dtype=dtype, device="cuda")
            n = lib.sb_lora_workspace_bytes(num_tokens, 128, width, 8, 3, fp32)
            work = torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda")  # its contents do not matter
            p = _C._ptr
            _lib.check(lib.sb_lora_linear(p(x), p(w), p(a), p(b), p(idx), 1, p(scale), p(room), fp32, num_tokens, 128,
                                          width, 8, 3, p(work), n, p(_C.device_status(x.device)), _C._stream()))
            assert bool((room[num_tokens:] == 7.0).all()) and bool((work[n:] == 0xA5).all())
            from sparsebench_b200 import lora_linear
            assert torch.equal(room[:num_tokens], lora_linear(x, w, a, b, idx, scale, dtype))
            assert lib.sb_lora_linear(p(x), p(w), p(a), p(b), p(idx), 1, p(scale), p(room), fp32, num_tokens, 128, width,
                                      8, 3, p(work), n - 1, None, ctypes.c_void_p(0)) == 1


@pytest.mark.parametrize("num_tokens", [3, 200])
def test_captured_call_and_another_stream(num_tokens):
    from sparsebench_b200 import lora_linear

    args = make(num_tokens, 256, 512, 16, 4, "any")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = lora_linear(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, lora_linear(*args))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = lora_linear(*args)
        again = lora_linear(args[0], *args[1:])  # two calls in one graph
    for seed in (5, 6):
        for dst, src in zip(args, make(num_tokens, 256, 512, 16, 4, "any", seed=seed)):
            dst.copy_(src)
        graph.replay()
        eager = lora_linear(*args)
        assert torch.equal(out, eager) and torch.equal(again, eager)


def test_router_logits_with_adapters_into_the_gated_layer():
    # As they are used together: the router's projection with each request's adapter -> picks and gates -> the experts.
    from oracle.gated import gated_reference
    from sparsebench_b200 import lora_linear, moe_forward_gated, route

    x, w, a, b, idx, scale = make(150, 256, 16, 8, 5)
    logits = lora_linear(x, w, a, b, idx, scale, out_dtype=torch.float32)
    picks, gates = route(logits, 2)
    value, bound = lora_reference(x, w, a, b, idx, scale, True)
    top = value.topk(3, dim=-1).values
    sure = (top[:, 1] - top[:, 2] > 4 * bound.amax(1)) & (top[:, 0] - top[:, 1] > 4 * bound.amax(1))
    assert int(sure.sum()) > 140 and torch.equal(picks[sure], value.topk(2, dim=-1).indices[sure])
    g = torch.Generator(device="cuda").manual_seed(1)
    wg, wu = ((torch.randn(16, 256, 384, generator=g, device="cuda") / 16).bfloat16() for _ in range(2))
    wd = (torch.randn(16, 384, 256, generator=g, device="cuda") / 384**0.5).bfloat16()
    out = moe_forward_gated(x, picks, gates, wg, wu, wd)
    want, tol = gated_reference(x, picks, gates, wg, wu, wd)["out"]
    assert bool(((out.double() - want).abs() <= 1.01 * (tol + 2.0**-8 * (want.abs() + tol))).all())


def test_empty_batch():
    from sparsebench_b200 import lora_linear

    assert lora_linear(*make(0, 64, 72, 8, 2)).shape == (0, 72)


def test_refusals():
    from sparsebench_b200 import lora_linear

    x, w, a, b, idx, scale = make(10, 64, 72, 8, 2)
    for args, text in [
        ((x.cpu(), w, a, b, idx), "CUDA tensor"),
        ((x.half(), w, a, b, idx), "bfloat16"),
        ((x, w.t().contiguous().t(), a, b, idx), "contiguous"),
        ((x, w[:32], a, b, idx), r"weight \[D, N\]"),
        ((x, w, a[:, :, :32].contiguous(), b, idx), "lora_a must be"),
        ((x, w, a, b[:1], idx), "lora_b"),
        ((x, w, a[:, :4].contiguous(), b[:, :4].contiguous(), idx), "rank"),
        ((x, w, a[:0], b[:0], idx), "number of adapters"),
        ((x, w, a, b, idx.float()), "int32 or int64"),
        ((x, w, a, b, idx[:5]), "int32 or int64"),
        ((x, w, a, b, idx.cpu()), "GPU"),
        ((x, w, a, b, idx, scale.double()), "float32"),
        ((x, w, a, b, idx, scale[:1]), "float32"),
        ((x, w, a, b, idx, scale, torch.float16), "out_dtype"),
        ((x[:, :60].contiguous(), w[:60].contiguous(), a[:, :, :60].contiguous(), b, idx), "multiple of 8"),
        ((x, w[:, :70].contiguous(), a, b[:, :, :70].contiguous(), idx), "multiple of 8"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            lora_linear(*args)
    odd = torch.empty(10 * 64 + 8, dtype=torch.bfloat16, device="cuda")[1:641].view(10, 64)
    with pytest.raises(RuntimeError, match="aligned"):
        lora_linear(odd, w, a, b, idx)
