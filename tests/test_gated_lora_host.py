"""What of the gated layer and the projection with adapters needs no GPU: their refusals, before anything is launched,
and their oracles against each other."""

import ctypes
import weakref

import pytest
import torch

from oracle.gated import activation, gated_layer, gated_reference, slope
from oracle.lora import lora_reference
from sparsebench_b200 import _build, _lib


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    _build.build()
    return _lib.load()


@pytest.mark.parametrize(("args", "text"), [
    ((0, 2, 128, 128, 4, 0), b"must be positive"),
    ((4, 0, 128, 128, 4, 0), b"must be positive"),
    ((4, 2, 64, 128, 4, 0), b"D (64) must be a positive multiple of 128"),
    ((4, 2, 128, 192, 4, 1), b"F (192) must be a positive multiple of 128"),
    ((4, 2, 128, 128, 0, 0), b""),
    ((4, 2, 128, 128, 1025, 0), b"num_experts"),
    ((2**31, 2, 128, 128, 4, 0), b"too large"),
    ((2**24, 8, 128, 2**20, 4, 1), b"too large"),
])
def test_gated_sizes_are_refused(lib, args, text) -> None:
    sizes = (ctypes.c_int64 * 3)()
    assert lib.sb_moe_gated_bytes(*args, sizes) == 1
    assert text in lib.sb_last_error()


def test_gated_sizes(lib) -> None:
    sizes = (ctypes.c_int64 * 3)()
    assert lib.sb_moe_gated_bytes(4096, 2, 1024, 4096, 64, 1, sizes) == 0
    rows = (8192 + 64 * 127) // 128 * 128
    blocks = rows * 4096 * 2
    assert sizes[0] > 3 * blocks + rows * 1024 * (2 + 4) and sizes[2] > 2 * blocks  # H, G, U, x and Y; dG, dU
    kept = list(sizes)
    assert lib.sb_moe_gated_bytes(4096, 2, 1024, 4096, 64, 0, sizes) == 0
    assert sizes[0] == 0 and blocks < sizes[1] < kept[0] and sizes[2] == 0
    assert lib.sb_moe_gated_bytes(32, 2, 1024, 4096, 64, 0, sizes) == 0  # a decoding step: H and Y of 64 copies
    assert sizes[1] == 64 * 4096 * 2 + 64 * 1024 * 4
    assert lib.sb_moe_gated_bytes(32, 2, 1024, 4096, 64, 0, None) == 1


def test_gated_calls_are_refused_before_any_launch(lib) -> None:
    one, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)  # never dereferenced
    big = 1 << 40

    def forward(x=one, ids=one, gate_dtype=0, state=one, scratch=one, act=0, state_bytes=big, scratch_bytes=big, d=128):
        return lib.sb_moe_gated_forward(x, ids, 1, one, gate_dtype, one, one, one, one, 100, 2, d, 128, 4, act, state,
                                        state_bytes, scratch, scratch_bytes, None, None)

    def backward(grad=one, gate_dtype=0, state=one, scratch=one, act=0, state_bytes=big, scratch_bytes=big):
        return lib.sb_moe_gated_backward(grad, one, gate_dtype, one, one, one, state, state_bytes, one, one, one, one, one,
                                         100, 2, 128, 128, 4, act, scratch, scratch_bytes, None, None)

    for call, text in [
        (lambda: forward(x=None), b"NULL"), (lambda: forward(ids=None), b"NULL"), (lambda: forward(scratch=None), b"NULL"),
        (lambda: forward(x=odd), b"aligned"), (lambda: forward(state=odd), b"aligned"), (lambda: forward(gate_dtype=2), b"gate_dtype"),
        (lambda: forward(act=2), b"activation"), (lambda: forward(d=130), b"multiple of 128"),
        (lambda: forward(state_bytes=1000), b"are needed"), (lambda: forward(scratch_bytes=0), b"are needed"),
        (lambda: backward(grad=None), b"NULL"), (lambda: backward(state=None), b"NULL"), (lambda: backward(grad=odd), b"aligned"),
        (lambda: backward(scratch=odd), b"aligned"), (lambda: backward(gate_dtype=-1), b"gate_dtype"), (lambda: backward(act=-1), b"activation"),
        (lambda: backward(state_bytes=1000), b"are needed"), (lambda: backward(scratch_bytes=1000), b"are needed"),
    ]:
        assert call() == 1 and text in lib.sb_last_error(), text
    args = [one] * 9
    assert lib.sb_sdd_gated(*args, 10, 128, 128, 4, 3, 5, 0, None, None) == 1 and b"activation" in lib.sb_last_error()
    assert lib.sb_sdd_gated(*args, 10, 100, 128, 4, 3, 0, 0, None, None) == 1 and b"multiple of 128" in lib.sb_last_error()
    assert lib.sb_sdd_gated(*args[:8], None, 10, 128, 128, 4, 3, 0, 0, None, None) == 1 and b"NULL" in lib.sb_last_error()
    assert lib.sb_sdd_gated(*args, 10, 128, 128, 4, 0, 0, 0, None, None) == 0  # no row blocks: nothing to do


def test_status_word_is_refused_without_a_place_for_it(lib) -> None:
    assert lib.sb_device_status_word(None) == 1 and b"NULL" in lib.sb_last_error()


@pytest.mark.parametrize(("sizes", "text"), [
    ((-1, 64, 64, 8, 2), b"31 bits"),
    ((10, 60, 64, 8, 2), b"D (60)"),
    ((10, 64, 60, 8, 2), b"N (60)"),
    ((10, 64, 64, 4, 2), b"rank (4)"),
    ((10, 64, 64, 136, 2), b"rank (136)"),
    ((10, 64, 64, 8, 0), b"adapters (0)"),
    ((10, 64, 64, 128, 2**25), b"31 bits"),
    ((10, 2**31 - 8, 64, 8, 2), b"D (2147483640) or N (64) is too large"),
    ((10, 64, 2**31 - 136, 8, 2), b"is too large"),
    ((65, 64, 2**27, 128, 2), b"the rank (128) times N (134217728) is too large"),
    ((100, 64, 2**28, 64, 2), b"times N"),
])
def test_lora_sizes_are_refused(lib, sizes, text) -> None:
    assert lib.sb_lora_workspace_bytes(*sizes, 0) == -1 and text in lib.sb_last_error()
    one = ctypes.c_void_p(1 << 20)
    assert lib.sb_lora_linear(one, one, one, one, one, 1, None, one, 0, *sizes, one, 1 << 40, None, None) == 1
    assert text in lib.sb_last_error()


def test_lora_calls_are_refused_before_any_launch(lib) -> None:
    one, odd = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 8)
    assert lib.sb_lora_linear(one, one, one, one, None, 1, None, one, 0, 10, 64, 64, 8, 2, one, 1 << 40, None, None) == 1
    assert b"NULL" in lib.sb_last_error()
    assert lib.sb_lora_linear(odd, one, one, one, one, 1, None, one, 0, 10, 64, 64, 8, 2, one, 1 << 40, None, None) == 1
    assert b"aligned" in lib.sb_last_error()
    assert lib.sb_lora_linear(one, one, one, one, one, 1, None, one, 0, 0, 64, 64, 8, 2, one, 0, None, None) == 0  # no tokens


def test_tensors_on_the_cpu_are_refused() -> None:
    from sparsebench_b200 import lora_linear, moe_forward_gated

    x, w = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(2, 128, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        moe_forward_gated(x, torch.zeros(4, 1, dtype=torch.int64), torch.ones(4, 1), w, w, w)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        lora_linear(x, w[0], torch.zeros(1, 8, 128, dtype=torch.bfloat16), torch.zeros(1, 8, 128, dtype=torch.bfloat16),
                    torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="w_down must be"):
        moe_forward_gated(x, torch.zeros(4, 1, dtype=torch.int64), torch.ones(4, 1), w, w, w[:1])


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated_oracle_against_autograd(act) -> None:
    g = torch.Generator().manual_seed(1)
    leaves = [torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()
              for s in ((9, 6), (9, 2), (4, 6, 5), (4, 6, 5), (4, 5, 6))]
    idx = torch.randint(-1, 5, (9, 2), generator=g)
    go = torch.randn(9, 6, generator=g, dtype=torch.float64)
    out = gated_layer(leaves[0], idx, *leaves[1:], act)
    grads = torch.autograd.grad(out, leaves, go)
    got = gated_reference(leaves[0].detach(), idx, *(t.detach() for t in leaves[1:]), act, go)
    torch.testing.assert_close(got["out"][0], out.detach(), rtol=1e-12, atol=1e-12)
    for name, want in zip(("dx", "dgate", "dw_gate", "dw_up", "dw_down"), grads):
        torch.testing.assert_close(got[name][0], want, rtol=1e-12, atol=1e-12)
        assert bool((got[name][1] >= 0).all())
    v = torch.linspace(-12, 12, 4001, dtype=torch.float64, requires_grad=True)
    (d,) = torch.autograd.grad(activation(v, act).sum(), v)
    torch.testing.assert_close(slope(v.detach(), act), d, rtol=1e-12, atol=1e-12)
    assert float(d.abs().max()) < 1.13  # what the error bounds take for the steepest slope


def test_lora_oracle_row_by_row() -> None:
    g = torch.Generator().manual_seed(2)
    x, w, a, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((7, 6), (6, 5), (3, 2, 6), (3, 2, 5)))
    idx = torch.tensor([0, 2, -1, 1, 3, 2, 0])
    scale = torch.tensor([0.5, 2.0, 1.5])
    got, bound = lora_reference(x, w, a, b, idx, scale)
    for t, i in enumerate(idx.tolist()):
        want = x[t] @ w
        if 0 <= i < 3:
            want = want + float(scale[i]) * ((a[i] @ x[t]) @ b[i])
        torch.testing.assert_close(got[t], want, rtol=1e-12, atol=1e-12)
    assert bool((bound > 0).all())


@pytest.fixture
def stand_in(monkeypatch):
    """The gated layer on the CPU with stand-ins for its two C calls: what Python does around them. Returns the list of
    (keep, weak reference to the state) of every forward call."""
    from sparsebench_b200 import _C

    calls = []

    def forward(x, idx, gate, w_gate, w_up, w_down, activation, keep):
        out = torch.empty_like(x)  # written by a kernel: nothing that autograd could follow
        out.detach().fill_(1)
        state = torch.zeros(1000, dtype=torch.uint8) if keep else None
        calls.append((keep, None if state is None else weakref.ref(state)))
        return out.detach(), state

    def backward(grad_out, x, gate, w_gate, w_up, w_down, state, activation, stream):
        assert stream == 77 and grad_out.is_contiguous() and grad_out.data_ptr() % 16 == 0
        assert state.dtype == torch.uint8 and state.numel() == 1000
        return tuple(torch.ones_like(t) for t in (x, gate, w_gate, w_up, w_down))

    monkeypatch.setattr(_C, "moe_gated_forward_cuda", forward)
    monkeypatch.setattr(_C, "moe_gated_backward_cuda", backward)
    monkeypatch.setattr(_C, "_raw_stream", lambda index: 77)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return calls


def gated_inputs() -> list[torch.Tensor]:
    w = torch.zeros(2, 128, 128, dtype=torch.bfloat16)
    return [torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(4, 1, dtype=torch.int64),
            torch.ones(4, 1, dtype=torch.bfloat16), w, w, w]


@pytest.mark.parametrize("which", [0, 2, 3, 4, 5])
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode_derivatives_are_refused(stand_in, which, leaf) -> None:
    from torch.autograd import forward_ad

    from sparsebench_b200 import moe_gated

    args = gated_inputs()
    with forward_ad.dual_level():
        dual = list(args)
        dual[which] = forward_ad.make_dual(args[which].clone().requires_grad_(leaf), torch.ones_like(args[which]))
        for mode in (torch.enable_grad, torch.no_grad):  # tangents do not ask for the gradient mode
            with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                moe_gated(*dual)
        assert not moe_gated(*args).requires_grad  # others in the same level: as ever
    primal = args[which]
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: moe_gated(*args[:which], t, *args[which + 1:]), (primal,), (torch.ones_like(primal),))
    assert [keep for keep, _ in stand_in] == [False]  # nothing was launched for the refused ones


def test_state_is_a_saved_tensor_of_autograd(stand_in) -> None:
    from torch.utils.checkpoint import checkpoint

    from sparsebench_b200 import moe_gated

    args = gated_inputs()
    args[0].requires_grad_()
    out = moe_gated(*args)
    keep, state = stand_in[-1]
    assert keep and state() is not None
    torch.autograd.grad(out, args[0], torch.ones_like(out), retain_graph=True)
    assert state() is not None
    out.backward(torch.ones_like(out))
    assert state() is None  # freed with the other saved tensors, though `out` and its graph are still here

    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(t.dtype), t.clone())[1], lambda t: t):
        out = moe_gated(*args)
    assert packed.count(torch.uint8) == 1 and stand_in[-1][1]() is None  # only what the hook made of it is left
    out.backward(torch.ones_like(out))

    before = len(stand_in)
    out = checkpoint(moe_gated, *args, use_reentrant=False)
    assert stand_in[-1][1]() is None  # nothing of the layer is kept until the backward pass runs the forward again
    out.backward(torch.ones_like(out))
    assert len(stand_in) == before + 2


def test_gradients_that_are_views_of_others_are_taken(stand_in) -> None:
    from sparsebench_b200 import moe_gated

    args = gated_inputs()
    args[0].requires_grad_()
    for front in (1, 8, 13):  # numbers in front of the layer's output in a larger vector
        out = moe_gated(*args)
        torch.cat([torch.zeros(front, dtype=torch.bfloat16), out.flatten()]).backward(torch.ones(front + 512, dtype=torch.bfloat16))
    moe_gated(*args).sum().backward()  # expanded
    moe_gated(*args).t().backward(torch.ones(128, 4, dtype=torch.bfloat16))  # transposed
    assert bool((args[0].grad == 5).all())
