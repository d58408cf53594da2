"""The gated MoE layer and its backward pass against their definitions in 64 bits (oracle/gated.py).

Two tolerances. Element by element: the bound that oracle/gated.py carries along (every rounding half a step, every
fp32 sum n 2^-24 of its magnitudes), with 1 % for products of two errors and the last rounding on top. Over a whole
output: roundings are independent and each is uniform within half a step, 2^-8 / sqrt(3) of the value in the root mean
square at most; a path has at most six of them (of G, U, H, w dO, dG or dU and the result), each passed on with a factor
of at most 1.13 (the largest slope of the activations), which makes sqrt(6) 1.13 2^-8 / sqrt(3) = 6.2e-3.
"""

import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from oracle.gated import gated_layer, gated_reference
from tests.cases import routing_case

pytestmark = pytest.mark.gpu

NORM_TOL = math.sqrt(6) * 1.13 * 2.0**-8 / math.sqrt(3)
NAMES = ("dx", "dgate", "dw_gate", "dw_up", "dw_down")


def make(num_tokens, d_model, ffn_dim, num_experts, k, seed=0, gate_dtype=torch.bfloat16, idx=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(num_tokens, d_model, generator=g).bfloat16()
    if idx is None:
        idx = torch.rand(num_tokens, num_experts, generator=g).topk(k, dim=-1).indices
    gate = torch.softmax(torch.randn(num_tokens, k, generator=g), dim=-1).to(gate_dtype)
    wg, wu = ((torch.randn(num_experts, d_model, ffn_dim, generator=g) / d_model**0.5).bfloat16() for _ in range(2))
    wd = (torch.randn(num_experts, ffn_dim, d_model, generator=g) / ffn_dim**0.5).bfloat16()
    go = torch.randn(num_tokens, d_model, generator=g).bfloat16()
    return [t.cuda() for t in (x, idx, gate, wg, wu, wd, go)]


def close(name, got, want, bound):
    assert torch.isfinite(got).all(), name
    last = (2.0**-8 if got.dtype == torch.bfloat16 else 2.0**-24)
    err = (got.double() - want).abs()
    # 2^-133 is half the smallest bf16 step: values that small round to it or to 0.
    allowed = 1.01 * (bound + last * (want.abs() + bound)) + 2.0**-133
    assert bool((err <= allowed).all()), f"{name}: {float((err / allowed).max()):.3g} times the bound"
    norm = float(want.norm())
    if norm > 0 and want.numel() >= 64:
        assert float(err.norm()) <= NORM_TOL * norm, f"{name}: {float(err.norm()) / norm:.3g} of the norm"


def step(x, idx, gate, wg, wu, wd, go, act):
    from sparsebench_b200 import moe_backward_gated, moe_forward_gated_saved

    out, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd, activation=act)
    return dict(zip(("out", *NAMES), (out, *moe_backward_gated(go, saved))))


def check(x, idx, gate, wg, wu, wd, go, act="silu"):
    from sparsebench_b200 import moe_forward_gated

    want = gated_reference(x, idx, gate, wg, wu, wd, act, go)
    got = step(x, idx, gate, wg, wu, wd, go, act)
    alone = moe_forward_gated(x, idx, gate, wg, wu, wd, activation=act)
    if idx.numel() <= 128:  # the decoding way, with another order of sums
        close("out", alone, *want["out"])
    else:
        assert torch.equal(got["out"], alone)
    for name, (value, bound) in want.items():
        assert got[name].dtype == (gate.dtype if name == "dgate" else torch.bfloat16)
        close(name, got[name], value, bound)
    return got


@pytest.mark.parametrize(("num_tokens", "d_model", "ffn_dim", "num_experts", "k", "act"), [
    (1, 128, 128, 1, 1, "silu"),
    (1, 256, 384, 8, 2, "gelu"),
    (2, 128, 640, 3, 3, "silu"),
    (63, 384, 256, 2, 1, "gelu"),
    (64, 256, 256, 4, 2, "silu"),
    (65, 128, 384, 1, 1, "silu"),
    (127, 640, 128, 3, 2, "gelu"),
    (129, 256, 512, 2, 2, "silu"),
    (300, 384, 896, 5, 4, "silu"),
    (513, 256, 1024, 8, 2, "gelu"),
    (1000, 512, 384, 64, 2, "silu"),
    (2049, 128, 256, 3, 2, "silu"),
    (700, 1024, 2048, 16, 1, "silu"),
])
def test_step_matches_definition(num_tokens, d_model, ffn_dim, num_experts, k, act):
    check(*make(num_tokens, d_model, ffn_dim, num_experts, k, seed=num_tokens), act=act)


@pytest.mark.parametrize("case", ["random", "zipf", "skewed", "two_experts_only", "empty_middle"])
def test_step_on_routing_patterns(case):
    idx = routing_case(case, 333, 8, seed=5)
    x, idx, gate, wg, wu, wd, go = make(333, 256, 384, 8, 2, idx=idx)
    got = check(x, idx, gate, wg, wu, wd, go)
    for e in range(8):
        if not bool((idx == e).any()):  # experts nobody picked get zeros, not what the memory held
            assert not any(bool(got[n][e].any()) for n in ("dw_gate", "dw_up", "dw_down"))


@pytest.mark.parametrize(("num_tokens", "d_model", "ffn_dim", "num_experts", "k"), [
    (1, 128, 128, 1, 1), (1, 1024, 4096, 64, 2), (1, 4096, 1408, 8, 2), (1, 128, 8192, 4, 4), (3, 640, 384, 5, 3),
    (8, 256, 1152, 2, 2), (16, 512, 512, 128, 4), (17, 384, 2048, 1, 1), (21, 1024, 256, 3, 3), (32, 256, 640, 40, 2),
    (33, 128, 256, 2, 1), (64, 512, 1024, 2, 1), (64, 2048, 128, 64, 1), (4, 256, 256, 16, 16), (43, 256, 384, 7, 2),
    (64, 384, 1152, 9, 2), (65, 128, 256, 3, 1), (128, 256, 512, 2, 1), (127, 128, 128, 130, 1), (32, 256, 256, 8, 4),
])
@pytest.mark.parametrize("pattern", ["spread", "one expert", "some out of range"])
def test_decoding_step(num_tokens, d_model, ffn_dim, num_experts, k, pattern):
    from sparsebench_b200 import moe_forward_gated

    x, idx, gate, wg, wu, wd, _ = make(num_tokens, d_model, ffn_dim, num_experts, k, seed=num_tokens + k)
    if pattern == "one expert":
        idx[:] = num_experts - 1
    elif pattern == "some out of range":
        idx[::2, 0] = -3
        idx[1::3] = num_experts
    for act, ids, g in (("silu", idx, gate), ("gelu", idx.int(), gate.float())):
        want = gated_reference(x, ids, g, wg, wu, wd, act)["out"]
        out = moe_forward_gated(x, ids, g, wg, wu, wd, activation=act)
        close("out", out, *want)
        assert torch.equal(out, moe_forward_gated(x, ids, g, wg, wu, wd, activation=act))


def test_decoding_step_captured_with_new_tokens_and_ids():
    from sparsebench_b200 import moe_forward_gated

    args = make(6, 256, 640, 8, 2)[:6]
    moe_forward_gated(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = moe_forward_gated(*args)
        second = moe_forward_gated(first, *args[1:])  # one layer on the other, twice the same weights
    for seed in (4, 5):
        for dst, src in zip(args, make(6, 256, 640, 8, 2, seed=seed)):
            dst.copy_(src)
        graph.replay()
        eager = moe_forward_gated(*args)
        assert torch.equal(first, eager) and torch.equal(second, moe_forward_gated(eager, *args[1:]))


def test_what_is_not_finite_in_an_expert_stays_with_its_tokens():
    from sparsebench_b200 import moe_forward_gated

    for num_tokens in (20, 200):
        x, idx, gate, wg, wu, wd, _ = make(num_tokens, 128, 256, 6, 2)
        want = moe_forward_gated(x, idx, gate, wg, wu, wd)
        others = (idx != 4).all(1)
        for which in range(3):
            broken = [t.clone() for t in (wg, wu, wd)]
            broken[which][4] = math.nan
            got = moe_forward_gated(x, idx, gate, *broken)
            assert torch.equal(got[others], want[others]) and got[~others].isnan().all()


def test_ids_out_of_range_and_the_same_expert_twice():
    x, idx, gate, wg, wu, wd, go = make(200, 128, 256, 6, 3)
    idx[::7, 0] = -1
    idx[3::11, 1] = 6
    idx[5::13] = idx[5::13, :1]  # one expert three times
    got = check(x, idx, gate, wg, wu, wd, go)
    assert not bool(got["dgate"][idx < 0].any()) and not bool(got["dgate"][idx == 6].any())
    idx[:] = 17  # nothing routed anywhere
    got = check(x, idx, gate, wg, wu, wd, go)
    assert not any(bool(t.any()) for t in got.values())


def test_ids_that_differ_in_their_upper_half_only():
    # 64-bit ids whose lower 32 bits name an expert are out of range all the same.
    for num_tokens in (20, 200):
        x, idx, gate, wg, wu, wd, go = make(num_tokens, 128, 256, 6, 2)
        idx[::5, 0] += 2**32
        idx[1::5, 1] -= 2**32
        idx[2::5, 0] += 2**40
        got = check(x, idx, gate, wg, wu, wd, go)
        assert not bool(got["dgate"][(idx < 0) | (idx >= 6)].any())


def test_int32_ids_and_fp32_gates():
    x, idx, gate, wg, wu, wd, go = make(150, 256, 256, 4, 2, gate_dtype=torch.float32)
    check(x, idx.int(), gate, wg, wu, wd, go)


def test_empty_batch():
    x, idx, gate, wg, wu, wd, go = make(0, 128, 256, 4, 2)
    got = step(x, idx, gate, wg, wu, wd, go, "silu")
    assert got["out"].shape == (0, 128) and got["dgate"].shape == (0, 2)
    assert got["dw_gate"].shape == wg.shape and not any(bool(t.any()) for t in got.values())


def test_gradients_against_differences():
    # Central differences of the definition in 64 bits along random directions. They are off by their step squared
    # (1e-8 of the third derivative); the kernel's gradient by NORM_TOL of its norm, in a random direction d of norm |d|
    # by NORM_TOL |grad| |d| at most.
    x, idx, gate, wg, wu, wd, go = make(90, 256, 384, 5, 2, seed=3)
    got = step(x, idx, gate, wg, wu, wd, go, "silu")
    leaves = [t.double() for t in (x, gate, wg, wu, wd)]
    g = torch.Generator(device="cuda").manual_seed(1)
    for i, name in enumerate(NAMES):
        d = torch.randn(leaves[i].shape, generator=g, device="cuda", dtype=torch.float64)
        sides = []
        for sign in (1, -1):
            moved = [t + sign * 1e-4 * d if n == i else t for n, t in enumerate(leaves)]
            out = gated_layer(moved[0], idx, *moved[1:], "silu")
            sides.append((out * go.double()).sum())
        slope = float(sides[0] - sides[1]) / 2e-4
        along = float((got[name].double() * d).sum())
        assert abs(along - slope) <= NORM_TOL * float(got[name].double().norm() * d.norm()) + 1e-5, name


def test_a_token_with_nan_or_inf_stays_alone():
    x, idx, gate, wg, wu, wd, go = make(140, 128, 256, 4, 2)
    want = step(x, idx, gate, wg, wu, wd, go, "silu")
    for bad in (math.nan, math.inf):
        y = x.clone()
        y[17, 3] = bad
        got = step(y, idx, gate, wg, wu, wd, go, "silu")
        others = torch.arange(140, device="cuda") != 17
        for n in ("out", "dx", "dgate"):
            assert torch.equal(got[n][others], want[n][others]), n
        untouched = [e for e in range(4) if e not in idx[17].tolist()]
        for n in ("dw_gate", "dw_up", "dw_down"):
            assert torch.equal(got[n][untouched], want[n][untouched]), n


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("which", ["w_gate", "w_up", "w_down"])
@pytest.mark.parametrize(("num_tokens", "d_model", "ffn_dim"), [(140, 128, 256), (70, 384, 640)])
def test_an_infinite_weight_comes_out_as_the_definition_has_it(num_tokens, d_model, ffn_dim, which, act):
    # Everything is positive, so no two infinities meet with opposite signs: what the definition makes infinite or NaN has
    # to be that, and all else finite. The rows of padding (0 times infinity) must not show.
    x, idx, gate, wg, wu, wd, go = (t if t.dtype == torch.int64 else t.abs() + 0.01 for t in make(num_tokens, d_model, ffn_dim, 4, 2))
    weights = {"w_gate": wg / 16, "w_up": wu / 16, "w_down": wd / 16}
    weights[which][1, 5, 9] = math.inf
    want = gated_reference(x, idx, gate, *weights.values(), act, go)
    got = step(x, idx, gate, *weights.values(), go, act)
    assert any(bool(torch.isinf(want[n][0][1]).any()) for n in ("dw_gate", "dw_up", "dw_down"))
    for name, (value, _) in want.items():
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(got[name]), kind(value)), (name, kind.__name__)


def test_memory_left_by_others_does_not_show():
    # Every buffer of the step is torch.empty: with the allocator's memory full of NaN the results are the same.
    args = make(210, 256, 384, 8, 2)
    first = step(*args, "gelu")
    torch.cuda.empty_cache()
    for size in (1 << 26, 1 << 22, 1 << 20, 1 << 18):
        junk = [torch.full((size,), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
        del junk
    again = step(*args, "gelu")
    for n in first:
        assert torch.equal(first[n], again[n]), n  # and run to run the same bits


def test_captured_step_and_another_stream():
    from sparsebench_b200 import moe_backward_gated, moe_forward_gated_saved

    x, idx, gate, wg, wu, wd, go = make(260, 256, 256, 8, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = step(x, idx, gate, wg, wu, wd, go, "silu")
    torch.cuda.current_stream().wait_stream(side)
    for n, t in step(x, idx, gate, wg, wu, wd, go, "silu").items():
        assert torch.equal(t, warm[n]), n
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd)
        grads = moe_backward_gated(go, saved)
    for seed in (7, 8):
        for dst, src in zip((x, idx, gate, wg, wu, wd, go), make(260, 256, 256, 8, 2, seed=seed)):
            dst.copy_(src)
        graph.replay()
        eager = step(x, idx, gate, wg, wu, wd, go, "silu")
        for n, t in zip(("out", *NAMES), (out, *grads)):
            assert torch.equal(t, eager[n]), n


FIRST_CALLS_UNDER_CAPTURE = """
import torch
from sparsebench_b200 import _C, lora_linear, moe_backward_gated, moe_forward, moe_forward_gated, moe_forward_gated_saved

g = torch.Generator(device="cuda").manual_seed(0)
n = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
x, wg, wu, wd, go = n(200, 256), n(4, 256, 512) / 16, n(4, 256, 512) / 16, n(4, 512, 256) / 20, n(200, 256)
idx, gate = torch.randint(0, 4, (200, 2), device="cuda"), torch.rand(200, 2, device="cuda").bfloat16()
w, a, b, ids = n(256, 264) / 16, n(3, 8, 256) / 16, n(3, 8, 264), torch.arange(200, device="cuda") % 4 - 1
told = []
real = _C._status_ptr
_C._status_ptr = lambda index: told.append(real(index)) or told[-1]

def calls():
    out, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd)
    return [lora_linear(x, w, a, b, ids), moe_forward_gated(x[:8], idx[:8], gate[:8], wg, wu, wd), out,
            *moe_backward_gated(go, saved), moe_forward(x, idx, gate, wg, wd)]

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = calls()
word = _C.device_status(torch.device("cuda", 0))
assert word.dtype == torch.int32 and word.shape == (1,) and word.device == x.device and int(word) == 0
assert len(told) >= 4 and set(told) == {word.data_ptr()}, (told, word.data_ptr())
word.fill_(4)  # what a wait that gave up would leave: it has to last
graph.replay()
torch.cuda.synchronize()
assert int(word) == 4
for p, q in zip(captured, calls()):
    assert torch.equal(p, q)
del captured, graph
torch.cuda.empty_cache()
junk = [torch.full((1 << s,), 7, dtype=torch.int32, device="cuda") for s in range(4, 24)]
assert int(word) == 4 and _C.device_status(x.device).data_ptr() == word.data_ptr()
print("as it should be")
"""


def test_first_calls_under_capture_report_to_the_status_word():
    # In a process of its own, whose first calls are captured: the kernels of the graph know the device's status word, which
    # is no part of the graph (neither set back by a replay nor handed out again with the graph's memory).
    root = Path(__file__).resolve().parent.parent
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS_UNDER_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "as it should be" in run.stdout, run.stdout[-1000:] + run.stderr[-3000:]


def test_autograd_form():
    from sparsebench_b200 import moe_gated

    x, idx, gate, wg, wu, wd, go = make(100, 128, 256, 4, 2)
    want = step(x, idx, gate, wg, wu, wd, go, "gelu")
    leaves = [t.clone().requires_grad_() for t in (x, gate, wg, wu, wd)]
    out = moe_gated(leaves[0], idx, *leaves[1:], activation="gelu")
    assert torch.equal(out, want["out"])
    grads = torch.autograd.grad(out, leaves, go, retain_graph=True)
    for n, g in zip(NAMES, grads):
        assert torch.equal(g, want[n]), n
    out.sum().backward()  # an expanded gradient, all its strides 0
    ones = step(x, idx, gate, wg, wu, wd, torch.ones_like(go), "gelu")
    for n, leaf in zip(NAMES, leaves):
        assert torch.equal(leaf.grad, ones[n]), n


def test_autograd_form_without_gradients_and_on_an_empty_batch():
    from sparsebench_b200 import moe_forward_gated, moe_gated

    x, idx, gate, wg, wu, wd, go = make(30, 128, 256, 4, 2)
    leaf = x.clone().requires_grad_()
    with torch.no_grad():
        out = moe_gated(leaf, idx, gate, wg, wu, wd)
    assert not out.requires_grad and torch.equal(out, moe_forward_gated(x, idx, gate, wg, wu, wd))
    assert not moe_gated(x, idx, gate, wg, wu, wd).requires_grad
    weight = wg.clone().requires_grad_()  # one leaf alone
    moe_gated(x, idx, gate, weight, wu, wd).backward(go)
    assert torch.equal(weight.grad, step(x, idx, gate, wg, wu, wd, go, "silu")["dw_gate"])
    empty = x[:0].clone().requires_grad_()
    moe_gated(empty, idx[:0], gate[:0], weight, wu, wd).sum().backward()
    assert empty.grad.shape == (0, 128)


def test_autograd_form_offloaded_and_checkpointed():
    from torch.utils.checkpoint import checkpoint

    from sparsebench_b200 import moe_gated

    x, idx, gate, wg, wu, wd, go = make(140, 256, 384, 4, 2)
    want = step(x, idx, gate, wg, wu, wd, go, "silu")
    leaves = [t.clone().requires_grad_() for t in (x, gate, wg, wu, wd)]
    call = lambda: moe_gated(leaves[0], idx, *leaves[1:])  # noqa: E731
    with torch.autograd.graph.save_on_cpu():
        offloaded = call()
    for out in (offloaded, checkpoint(call, use_reentrant=False)):
        assert torch.equal(out, want["out"])
        for n, g in zip(NAMES, torch.autograd.grad(out, leaves, go)):
            assert torch.equal(g, want[n]), n
    before = torch.cuda.memory_allocated()
    out = call()
    state = torch.cuda.memory_allocated() - before - out.numel() * 2
    grads = torch.autograd.grad(out, leaves, go)
    left = torch.cuda.memory_allocated() - before - out.numel() * 2 - sum(g.numel() * 2 for g in grads)
    assert state > 6 * 128 * 4 * (256 + 384) and left < state / 4  # rows * (6 D + 6 F) bytes, freed while `out` is alive


def test_backward_twice_and_two_forwards_at_once():
    from sparsebench_b200 import moe_backward_gated, moe_forward_gated_saved

    a, b = make(140, 256, 384, 8, 2, seed=1), make(77, 256, 384, 8, 2, seed=2)
    want = [step(*args, "silu") for args in (a, b)]
    _, first = moe_forward_gated_saved(*a[:6])
    _, second = moe_forward_gated_saved(*b[:6])
    for _ in range(2):
        for saved, args, ref in ((first, a, want[0]), (second, b, want[1])):
            for n, g in zip(NAMES, moe_backward_gated(args[6], saved)):
                assert torch.equal(g, ref[n]), n


def test_views_with_an_offset_and_misaligned_ones():
    from sparsebench_b200 import moe_forward_gated

    x, idx, gate, wg, wu, wd, _ = make(100, 128, 256, 4, 2)
    for num_tokens in (10, 90):
        want = moe_forward_gated(x[:num_tokens].clone(), idx[:num_tokens].clone(), gate[:num_tokens].clone(), wg, wu, wd)
        stack = torch.stack([wg, wg])  # a layer's weights as a slice of all layers'
        got = moe_forward_gated(x[:num_tokens], idx[:num_tokens], gate[:num_tokens], stack[1], wu, wd)
        assert torch.equal(got, want)
        odd = torch.empty(num_tokens * 128 + 8, dtype=torch.bfloat16, device="cuda")[1:num_tokens * 128 + 1].view(num_tokens, 128)
        odd.copy_(x[:num_tokens])
        with pytest.raises(RuntimeError, match="aligned"):
            moe_forward_gated(odd, idx[:num_tokens], gate[:num_tokens], wg, wu, wd)


def test_state_outlives_a_backward_on_another_stream():
    # The backward call waits on its stream behind 50 ms of nothing; meanwhile the last reference to the state goes, and the
    # forward's stream asks for memory of that size. It must not get the state's.
    from sparsebench_b200 import moe_backward_gated, moe_forward_gated_saved

    x, idx, gate, wg, wu, wd, go = make(400, 256, 512, 4, 2)
    want = step(x, idx, gate, wg, wu, wd, go, "silu")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        moe_backward_gated(go, moe_forward_gated_saved(x, idx, gate, wg, wu, wd)[1])  # warm: memory of that stream
    torch.cuda.synchronize()
    _, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd)
    where, size = saved.state.data_ptr(), saved.state.numel()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        grads = moe_backward_gated(go, saved)
        done = torch.cuda.Event()
        done.record()
    del saved
    junk = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert not done.query()  # else this shows nothing
    assert all(not where <= t.data_ptr() < where + size for t in junk)
    torch.cuda.synchronize()
    for n, g in zip(NAMES, grads):
        assert torch.equal(g, want[n]), n


def test_backward_captured_alone():
    # An eager forward's state read by a graph of the backward call, on the capture's stream; then eager steps again.
    from sparsebench_b200 import moe_backward_gated, moe_forward_gated_saved

    x, idx, gate, wg, wu, wd, go = make(260, 256, 384, 4, 2)
    _, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = moe_backward_gated(go, saved)
    for seed in (1, 2):
        go.copy_(make(260, 256, 384, 4, 2, seed=seed)[6])
        graph.replay()
        want = step(x, idx, gate, wg, wu, wd, go, "silu")
        for n, g in zip(NAMES, grads):
            assert torch.equal(g, want[n]), n
    del graph, grads, saved  # the state's memory goes back to the allocator behind the capture's stream
    torch.cuda.empty_cache()
    again = step(x, idx, gate, wg, wu, wd, go, "silu")
    for n in again:
        assert torch.equal(again[n], want[n]), n


def test_two_streams_at_once():
    from sparsebench_b200 import lora_linear, moe_forward_gated

    args = [make(t, 256, 512, 8, 2, seed=t) for t in (4, 300)]
    g = torch.Generator(device="cuda").manual_seed(3)
    w = (torch.randn(256, 264, generator=g, device="cuda") / 16).bfloat16()
    la = (torch.randn(3, 16, 256, generator=g, device="cuda") / 16).bfloat16()
    lb = torch.randn(3, 16, 264, generator=g, device="cuda").bfloat16()
    ids = [torch.arange(t, device="cuda") % 4 - 1 for t in (4, 300)]
    run = lambda i: (moe_forward_gated(*args[i][:6]), lora_linear(args[i][0], w, la, lb, ids[i]))  # noqa: E731
    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for round_ in range(20):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((n % 2, run(n % 2)))
    torch.cuda.synchronize()
    for i, (out, y) in got:
        assert torch.equal(out, want[i][0]) and torch.equal(y, want[i][1])


def test_rows_past_two_to_the_31_values():
    # 132 000 tokens x 16 384 columns are 2.16e9 values of x, of Y and of their gradients (routing itself refuses blocks of
    # H with more than 2^31). Checked on the last tokens, which lie behind the 2^31st value.
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("needs 70 GB of free memory")
    num_tokens, d_model, ffn_dim, experts = 132_000, 16_384, 128, 2
    g = torch.Generator(device="cuda").manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    x, go = normal(num_tokens, d_model), normal(num_tokens, d_model)
    idx = (torch.arange(num_tokens, device="cuda") % 2)[:, None].contiguous()
    gate = torch.rand(num_tokens, 1, generator=g, device="cuda").bfloat16()
    wg, wu = (normal(experts, d_model, ffn_dim) * d_model**-0.5 for _ in range(2))
    wd = normal(experts, ffn_dim, d_model) * ffn_dim**-0.5
    got = step(x, idx, gate, wg, wu, wd, go, "silu")
    last = slice(num_tokens - 40, num_tokens)
    want = gated_reference(x[last], idx[last], gate[last], wg, wu, wd, "silu", go[last])
    for name in ("out", "dx", "dgate"):
        close(name, got[name][last], *want[name])
    del x, go, got
    torch.cuda.empty_cache()


def test_sdd_gated_on_a_trimmed_topology():
    from sparsebench_b200 import route_device, sdd_gated

    x, idx, gate, wg, wu, wd, go = make(150, 128, 256, 4, 2)
    topo = route_device(idx, 4, 256, 128)
    trimmed = topo.to_topology()
    h = sdd_gated(x, wg, wu, trimmed, activation="gelu")
    assert h.shape == (trimmed.col_indices.numel(), 128, 128)
    assert torch.equal(h, sdd_gated(x, wg, wu, topo, activation="gelu")[:h.shape[0]])
    none = route_device(torch.full_like(idx, 9), 4, 256, 128).to_topology(check=False)
    assert sdd_gated(x, wg, wu, none).shape == (0, 128, 128)
    with pytest.raises(ValueError, match="block size 128"):
        sdd_gated(x, wg, wu, route_device(idx, 4, 256, 64))


def test_sdd_gated_with_the_layout_of_a_larger_batch():
    # x ends where memory that must not be read begins: tokens it does not have are zeros.
    from sparsebench_b200 import route_device, sdd_gated

    x, idx, gate, wg, wu, wd, go = make(300, 128, 256, 4, 2)
    topo = route_device(idx, 4, 256, 128)
    behind = torch.where((torch.arange(300, device="cuda") < 180)[:, None], x, torch.zeros_like(x))
    want = sdd_gated(behind, wg, wu, topo)
    live = int(topo.padded_offsets[-1]) // 128 * 2  # blocks of live row blocks
    assert torch.equal(sdd_gated(x[:180].clone(), wg, wu, topo)[:live], want[:live])


def test_sdd_gated_alone():
    from sparsebench_b200 import route_device, sdd_gated

    x, idx, gate, wg, wu, wd, go = make(180, 128, 384, 4, 2)
    topo = route_device(idx, 4, 384, 128)
    h = sdd_gated(x, wg, wu, topo)
    trimmed = topo.to_topology()
    for rb, e in enumerate(trimmed.row_block_expert.tolist()):
        token = trimmed.row_token[rb * 128:(rb + 1) * 128].long()
        rows = torch.where((token >= 0)[:, None], x[token.clamp(min=0)], torch.zeros((), device="cuda", dtype=x.dtype)).double()
        g, u = rows @ wg[e].double(), rows @ wu[e].double()
        want = g / (1 + torch.exp(-g)) * u
        got = torch.cat(list(h[rb * 3:(rb + 1) * 3]), dim=1)
        bound = 2.0**-8 * want.abs() + 128 * 2.0**-24 * 4 * (rows.abs() @ wg[e].double().abs() + 1) * (rows.abs() @ wu[e].double().abs() + 1)
        assert bool(((got.double() - want).abs() <= bound).all())
        assert not bool(got[token < 0].any())


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_backward_keeps_what_is_not_finite_in_an_expert_to_itself(which, bad):
    # D and F are odd multiples of 128: tiles of 256 columns reach into the next expert's weights and the next row block's
    # hidden gradients, and row blocks of few rows leave the rest of a stage as it was. Expert 4 is neither the first nor last.
    x, idx, gate, wg, wu, wd, go = make(200, 384, 640, 6, 2)
    idx[idx[:, 0] == 2, 0] = 4  # expert 4 has more than a row block's half, expert 2 few rows
    want = step(x, idx, gate, wg, wu, wd, go, "silu")
    weights = [t.clone() for t in (wg, wu, wd)]
    weights[which][4] = bad
    got = step(x, idx, gate, *weights, go, "silu")
    others = (idx != 4).all(1)
    assert 20 < int(others.sum()) < 180
    for n in ("out", "dx"):
        assert torch.equal(got[n][others], want[n][others]), n
    assert torch.equal(got["dgate"][idx != 4], want["dgate"][idx != 4])
    for n in ("dw_gate", "dw_up", "dw_down"):
        for e in (0, 1, 2, 3, 5):
            assert torch.equal(got[n][e], want[n][e]), (n, e)
    assert not torch.isfinite(got["out"][~others]).any()
    assert not all(bool(torch.isfinite(got[n][4]).all()) for n in ("dw_gate", "dw_up", "dw_down"))


@pytest.mark.parametrize("gate_dtype", [torch.bfloat16, torch.float32])
def test_gates_of_zero_have_gradients(gate_dtype):
    # dgate = dO . Y does not pass through the gate; everything else of such a copy is exactly 0.
    x, idx, gate, wg, wu, wd, go = make(150, 256, 384, 5, 2, seed=4, gate_dtype=gate_dtype)
    gate[::3, 0] = 0
    gate[1::7] = 0
    gate[2::9, 1] = -0.0
    got = check(x, idx, gate, wg, wu, wd, go)
    assert bool((got["dgate"][gate == 0] != 0).all())
    gone = (gate == 0).all(1)
    assert int(gone.sum()) > 10 and not bool(got["dx"][gone].any()) and not bool(got["out"][gone].any())
    got = check(x, idx, torch.zeros_like(gate), wg, wu, wd, go, "gelu")
    assert not any(bool(got[n].any()) for n in ("out", "dx", "dw_gate", "dw_up", "dw_down"))


@pytest.mark.parametrize("skip", [False, True])
@pytest.mark.parametrize(("num_tokens", "d_model", "ffn_dim", "num_experts", "k"),
                         [(1, 256, 128, 3, 2), (150, 256, 640, 4, 2), (700, 512, 256, 9, 3)])
def test_sdd_gated_then_dsd_then_combine(num_tokens, d_model, ffn_dim, num_experts, k, skip):
    # The layer from its parts. Between dsd and combine a row is bf16: half a step of every copy's share on top of the bound.
    from sparsebench_b200 import combine, dsd, route_device, sdd_gated

    x, idx, gate, wg, wu, wd, _ = make(num_tokens, d_model, ffn_dim, num_experts, k, seed=9)
    topo = route_device(idx, num_experts, ffn_dim, 128)
    h = sdd_gated(x, wg, wu, topo, activation="gelu", skip_padding_rows=skip)
    y = dsd(h, wd.reshape(-1, d_model), topo, skip_padding_rows=skip)
    out = combine(y, gate, topo)
    want, bound = gated_reference(x, idx, gate, wg, wu, wd, "gelu")["out"]
    for j in range(k):
        share, off = gated_reference(x, idx[:, j:j + 1], gate[:, j:j + 1], wg, wu, wd, "gelu")["out"]
        bound = bound + 2.0**-8 * (share.abs() + off)
    err = (out.double() - want).abs()
    assert bool((err <= 1.01 * (bound + 2.0**-8 * (want.abs() + bound)) + 2.0**-133).all())


def test_refusals():
    from sparsebench_b200 import moe_backward_gated, moe_forward_gated, moe_forward_gated_saved

    x, idx, gate, wg, wu, wd, go = make(20, 128, 256, 4, 2)
    for args, text in [
        ((x, idx, gate, wg, wu[:, :, :128], wd), "w_gate and w_up"),
        ((x, idx, gate, wg, wu, wd[:, :128]), "w_down must be"),
        ((x[:, :64], idx, gate, wg, wu, wd), r"\[T, D\]"),
        ((x, idx[:10], gate, wg, wu, wd), r"\[T, k\]"),
    ]:
        with pytest.raises(ValueError, match=text):
            moe_forward_gated(*args)
    wide = torch.empty(4, 128, 192, dtype=torch.bfloat16, device="cuda")
    for args, kwargs, text in [
        ((x.half(), idx, gate, wg, wu, wd), {}, "bfloat16"),
        ((x, idx, gate, wg.float(), wu, wd), {}, "bfloat16"),
        ((x.cpu(), idx, gate, wg, wu, wd), {}, "CUDA tensor"),
        ((x, idx.cpu(), gate, wg, wu, wd), {}, "same GPU"),
        ((x, idx, gate, wg.transpose(1, 2).contiguous().transpose(1, 2), wu, wd), {}, "contiguous"),
        ((x, idx, gate, wide, wide, wide.transpose(1, 2).contiguous()), {}, "multiple of 128"),
        ((x, idx, gate, wg, wu, wd), {"activation": "relu"}, "activation"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            moe_forward_gated(*args, **kwargs)
    _, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd)
    with pytest.raises(ValueError, match="grad_out"):
        moe_backward_gated(go[:10], saved)
    with pytest.raises(RuntimeError, match="grad_out must be bfloat16"):
        moe_backward_gated(go.float(), saved)
    with pytest.raises(RuntimeError, match="contiguous"):
        moe_backward_gated(go[:1].expand(20, 128), saved)


def test_backward_refuses_what_is_not_what_the_forward_kept():
    # saved_tensors_hooks and dataclasses.replace can put other tensors there; none of these may reach a kernel.
    from dataclasses import replace

    from sparsebench_b200 import moe_backward_gated, moe_forward_gated_saved, moe_gated

    x, idx, gate, wg, wu, wd, go = make(20, 128, 256, 4, 2)
    _, saved = moe_forward_gated_saved(x, idx, gate, wg, wu, wd)
    for change, error, text in [
        ({"w_up": wu.cpu()}, RuntimeError, "w_up must be a CUDA tensor"),
        ({"w_down": wd.float()}, RuntimeError, "w_down must be bfloat16"),
        ({"w_gate": wg.transpose(1, 2).contiguous().transpose(1, 2)}, RuntimeError, "w_gate must be contiguous"),
        ({"w_up": wu[:3]}, ValueError, "w_gate and w_up"),
        ({"w_down": wd[:, :128]}, ValueError, "w_down must be"),
        ({"expert_weight": gate[:10]}, ValueError, r"\[T, k\]"),
        ({"expert_weight": gate.cpu()}, RuntimeError, "expert_weight is on cpu"),
        ({"expert_weight": gate.half()}, RuntimeError, "bfloat16 or float32"),
        ({"state": saved.state.cpu()}, RuntimeError, "state is on cpu"),
        ({"state": saved.state[:-256]}, RuntimeError, "are needed"),
        ({"state": saved.state.float()}, RuntimeError, "uint8"),
        ({"activation": "relu"}, RuntimeError, "activation"),
        ({"x": x.cpu()}, RuntimeError, "CUDA|same GPU"),
    ]:
        with pytest.raises(error, match=text):
            moe_backward_gated(go, replace(saved, **change))
    leaf = x.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):  # never brought back
        out = moe_gated(leaf, idx, gate, wg, wu, wd)
    with pytest.raises(RuntimeError):
        out.backward(go)
    assert torch.equal(moe_backward_gated(go, saved).x, step(x, idx, gate, wg, wu, wd, go, "silu")["dx"])


def test_autograd_backward_refuses_capture():
    from sparsebench_b200 import moe_gated

    x, idx, gate, wg, wu, wd, go = make(20, 128, 128, 2, 1)
    leaf = x.clone().requires_grad_()
    out = moe_gated(leaf, idx, gate, wg, wu, wd)

    class Ctx:  # what the node hands its backward; the refusal comes before anything is launched or read
        pass

    from sparsebench_b200 import gated

    real = torch.cuda.is_current_stream_capturing
    torch.cuda.is_current_stream_capturing = lambda: True
    try:
        with pytest.raises(RuntimeError, match="moe_backward_gated"):
            gated._GatedMoE.backward(Ctx(), go)
    finally:
        torch.cuda.is_current_stream_capturing = real
    assert out.requires_grad
