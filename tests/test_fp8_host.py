"""What the block-scaled FP8 products and the group-limited router refuse,
without a GPU (fake CUDA tensors; nothing is launched)."""

from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch
from conftest import pkg
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

BF16 = torch.bfloat16
F8 = torch.float8_e4m3fn


def cuda(*shape, dtype=BF16):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def weight(*shape):
    n, k = shape[-2:]
    return cuda(*shape, dtype=F8), cuda(*shape[:-2], -(-n // 128), -(-k // 128), dtype=torch.float32)


@pytest.mark.parametrize("kw", [
    dict(groups=3, top_groups=1), dict(groups=4), dict(groups=4, top_groups=5), dict(groups=4, top_groups=0),
    dict(groups=0, top_groups=1), dict(groups=64, top_groups=1), dict(top_groups=2),
    dict(groups=16, top_groups=1), dict(groups=4, top_groups=2, group_score="mean"),
])
def test_route_refuses_bad_groups(kw):
    with FakeTensorMode(), pytest.raises(ValueError):
        pkg().ops.route(cuda(5, 64, dtype=torch.float32), None, 6, "sigmoid", **kw)


def test_route_refuses_bad_arguments():
    with FakeTensorMode():
        logits = cuda(5, 64, dtype=torch.float32)
        for args in ((logits, None, 4, "tanh"), (logits, None, 0, "sigmoid"), (logits, None, 65, "sigmoid"),
                     (logits, cuda(63, dtype=torch.float32), 4, "sigmoid"), (logits.to(BF16), None, 4, "sigmoid")):
            with pytest.raises(ValueError):
                pkg().ops.route(*args, groups=4, top_groups=2)


@pytest.mark.parametrize("kind", ["dtype", "width", "columns", "scale_shape", "scale_dtype", "weight_dtype",
                                  "weight_strided", "cpu", "transposed", "pitch"])
def test_linear_refuses(kind):
    with FakeTensorMode():
        x, (q, s) = cuda(4, 256), weight(300, 256)
        if kind == "dtype":
            x = x.float()
        elif kind == "width":
            x = cuda(4, 128)
        elif kind == "columns":
            x = cuda(4, 512)[:, ::2]
        elif kind == "scale_shape":
            s = s[:2].contiguous()
        elif kind == "scale_dtype":
            s = s.to(BF16)
        elif kind == "weight_dtype":
            q = q.to(BF16)
        elif kind == "weight_strided":
            q = cuda(256, 300, dtype=F8).T
        elif kind == "cpu":
            x = torch.empty(4, 256, dtype=BF16)
        elif kind == "transposed":
            x = cuda(256, 4).T
        else:
            x = cuda(4, 260)[:, :256]  # rows 260 elements apart are not 16-byte aligned
        with pytest.raises(ValueError):
            pkg().ops.fp8_linear(x, q, s)


def test_products_refuse_gradients():
    with FakeTensorMode():
        q, s = weight(128, 256)
        with pytest.raises(RuntimeError, match="inference"):
            pkg().ops.fp8_linear(cuda(4, 256).requires_grad_(), q, s)
        with pytest.raises(RuntimeError, match="inference"):
            pkg().ops.fp8_linear(cuda(4, 256), q, s.requires_grad_())


@pytest.mark.parametrize("which", ["residual", "norm_weight", "mod", "shared"])
def test_tail_refuses_gradients(which):
    """The fused tail's outputs carry no gradient, so no input of it may want one."""
    with FakeTensorMode():
        e, c, f, t, k = 4, 256, 128, 6, 2
        given = dict(residual=cuda(t, c), norm_weight=cuda(c, dtype=torch.float32), mod=cuda(t, 2 * c), shared=cuda(t, c))
        given[which].requires_grad_()
        shared = given.pop("shared")
        with pytest.raises(RuntimeError, match="inference"):
            pkg().ops.fp8_moe_forward(cuda(t, c), cuda(t, k, dtype=torch.int64), cuda(t, k), *weight(e, 2 * f, c),
                                      *weight(e, c, f), 1.0, shared, tail=pkg().ops.Tail(**given))


def test_quantizers_refuse_gradients():
    with FakeTensorMode():
        with pytest.raises(RuntimeError, match="inference"):
            pkg().ops.fp8_quantize(cuda(4, 256).requires_grad_())
        with pytest.raises(RuntimeError, match="inference"):
            pkg().ops.fp8_pack_weights(cuda(256, 128).requires_grad_())


@pytest.mark.parametrize("kind", ["odd", "small", "down", "out", "x_strided", "experts"])
def test_mlp_refuses(kind):
    with FakeTensorMode():
        c, f = 256, 384
        x, gu, down, out = cuda(4, c), weight(2 * f, c), weight(c, f), None
        if kind == "odd":
            gu = weight(2 * f + 1, c)
        elif kind == "small":
            gu, down = weight(2 * 64, c), weight(c, 64)
        elif kind == "down":
            down = weight(c, 256)
        elif kind == "out":
            out = cuda(3, c)
        elif kind == "x_strided":
            x = cuda(4, 2 * c)[:, :c]
        else:
            gu, down = weight(2, 2 * f, c), weight(2, c, f)
        with pytest.raises(ValueError):
            pkg().ops.fp8_mlp(x, *gu, *down, out=out)


@pytest.mark.parametrize("kind", ["top_dtype", "top_k", "gate_shape", "gate_dtype", "shared", "tokens", "width", "out"])
def test_moe_forward_refuses(kind):
    with FakeTensorMode():
        e, c, f, t, k = 4, 256, 128, 6, 2
        x, top, gate, shared, out = cuda(t, c), cuda(t, k, dtype=torch.int64), cuda(t, k), None, None
        if kind == "top_dtype":
            top = top.to(torch.int32)
        elif kind == "top_k":
            top, gate = cuda(t, 5, dtype=torch.int64), cuda(t, 5)
        elif kind == "gate_shape":
            gate = cuda(t, 1)
        elif kind == "gate_dtype":
            gate = gate.float()
        elif kind == "shared":
            shared = cuda(t, 128)
        elif kind == "tokens":
            x = cuda(t + 1, c)
        elif kind == "width":
            x = cuda(t, 128)
        else:
            out = cuda(t, c, dtype=torch.float32)
        with pytest.raises(ValueError):
            pkg().ops.fp8_moe_forward(x, top, gate, *weight(e, 2 * f, c), *weight(e, c, f), 1.0, shared, out=out)


def packed(e=2, c=128, f=128):
    return {
        "gate_up_q": torch.zeros(e, 2 * f, c).to(F8), "gate_up_scale": torch.ones(e, 2 * f // 128, c // 128),
        "down_q": torch.zeros(e, c, f).to(F8), "down_scale": torch.ones(e, c // 128, f // 128),
    }


@pytest.mark.parametrize("kind", ["missing", "extra", "shape", "dtype", "scale_nan", "scale_zero", "value_nan", "odd"])
def test_bank_rejects_corrupt_state(kind):
    state = packed()
    if kind == "missing":
        del state["down_q"]
    elif kind == "extra":
        state["bias"] = torch.ones(1)
    elif kind == "shape":
        state["down_q"] = state["down_q"][:, :, :64].contiguous()
    elif kind == "dtype":
        state["down_scale"] = state["down_scale"].to(BF16)
    elif kind.startswith("scale"):
        state["gate_up_scale"][0, 0, 0] = float("nan") if kind == "scale_nan" else 0.0
    elif kind == "value_nan":
        state["gate_up_q"].view(torch.uint8)[0, 0, 0] = 0xFF
    else:
        state = packed(c=192)
    with pytest.raises(ValueError):
        pkg().B200FP8RoutedExperts.from_packed(state)


def test_bank_validation_needs_no_copies_of_the_bank():
    """The search for NaN codes goes through the bank in pieces, and finds one in
    the last of them."""
    class Largest(TorchDispatchMode):
        nbytes = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            given = {a.untyped_storage().data_ptr() for a in args if isinstance(a, torch.Tensor)}
            if isinstance(out, torch.Tensor) and out.untyped_storage().data_ptr() not in given:
                self.nbytes = max(self.nbytes, out.nbytes)
            return out

    state = packed(e=3, c=4096, f=4096)
    with Largest() as largest:
        pkg().B200FP8RoutedExperts.from_packed(state)
    assert largest.nbytes <= 2**24 < state["gate_up_q"].nbytes // 4
    state["gate_up_q"].view(torch.uint8)[-1, -1, -1] = 0x7F
    with pytest.raises(ValueError, match="E4M3"):
        pkg().B200FP8RoutedExperts.from_packed(state)


def test_bank_is_inference_only_and_keeps_its_types():
    bank = pkg().B200FP8RoutedExperts.from_packed(packed())
    assert bank.to("cpu") is bank and not bank.training
    with pytest.raises(TypeError, match="casts"):
        bank.to(BF16)
    with pytest.raises(RuntimeError, match="inference"):
        bank.train()
    x, top, gate = torch.ones(3, 128, dtype=BF16), torch.zeros(3, 1, dtype=torch.int64), torch.ones(3, 1, dtype=BF16)
    with pytest.raises(ValueError, match="CUDA"):
        bank.routed_forward(x, top, gate, scaling=1.0, chunk_size=2)
    with pytest.raises(RuntimeError, match="inference"):
        bank.routed_forward(x.requires_grad_(), top, gate, scaling=1.0, chunk_size=2)
    for kw in (dict(scaling=float("nan"), chunk_size=2), dict(scaling=1.0, chunk_size=0)):
        with pytest.raises(ValueError):
            bank.routed_forward(x.detach(), top, gate, **kw)
    assert set(bank.state_dict()) == set(packed())
    again = pkg().B200FP8RoutedExperts.from_packed({k: v.clone() for k, v in bank.state_dict().items()})
    assert (again.num_experts, again.in_features, again.hidden_features) == (2, 128, 128)


@pytest.mark.parametrize("kind,tail", [
    *((kind, tail) for kind in ("top_more", "top_fewer", "gate_more", "gate_k", "x_3d") for tail in (False, True)),
    ("shared", True), ("shared_dtype", True),  # without a tail such a shared output is added by torch
])
def test_bank_checks_the_whole_call_before_it_is_cut_in_chunks(monkeypatch, kind, tail):
    """Rows behind the last token's must not vanish in the slices of the chunks."""
    called = []
    monkeypatch.setattr(pkg().ops, "fp8_moe_forward", lambda *a, **kw: called.append(1))
    bank = pkg().B200FP8RoutedExperts.from_packed(packed())
    t = 5
    x, shared, residual = (torch.ones(t, 128, dtype=BF16) for _ in range(3))
    top, gate = torch.zeros(t, 2, dtype=torch.int64), torch.ones(t, 2, dtype=BF16)
    if kind == "shared":
        shared = torch.ones(t + 3, 128, dtype=BF16)
    elif kind == "shared_dtype":
        shared = shared.float()
    elif kind == "top_more":
        top = torch.zeros(t + 3, 2, dtype=torch.int64)
    elif kind == "top_fewer":
        top, gate = top[:4], gate[:4]
    elif kind == "gate_more":
        gate = torch.ones(t + 3, 2, dtype=BF16)
    elif kind == "gate_k":
        gate = gate[:, :1]
    else:
        x = residual = torch.ones(t, 1, 128, dtype=BF16)
    with pytest.raises(ValueError):
        if tail:
            bank.routed_forward_tail(x, top, gate, scaling=1.0, chunk_size=2, tail=pkg().ops.Tail(residual),
                                     shared=shared)
        else:
            bank.routed_forward(x, top, gate, scaling=1.0, chunk_size=2)
    assert not called


def test_the_tail_function_takes_either_bank(monkeypatch):
    """``praxis_b200.routed_forward_tail`` runs an FP8 bank's own tail."""
    rows = []

    def fake(x, *args, tail, tail_out, **kwargs):
        rows.append(x.shape[0])
        tail_out[0].copy_(tail.residual)

    monkeypatch.setattr(pkg().ops, "fp8_moe_forward", fake)
    bank = pkg().B200FP8RoutedExperts.from_packed(packed())
    x, residual = torch.ones(5, 128, dtype=BF16), torch.randn(5, 128).to(BF16)
    new, normed = pkg().routed_forward_tail(
        bank, x, torch.zeros(5, 2, dtype=torch.int64), torch.ones(5, 2, dtype=BF16), scaling=1.0, chunk_size=2,
        tail=pkg().ops.Tail(residual), shared=x)
    assert rows == [2, 2, 1] and torch.equal(new, residual) and normed is None


def test_module_takes_groups_and_formats():
    M = pkg().B200MoEFeedForward
    m = M(128, 128, 16, 4, router_groups=4, router_top_groups=2)
    assert (m.router_groups, m.router_top_groups, m.router_group_score) == (4, 2, "top2")
    for kw in (dict(router_groups=3, router_top_groups=1), dict(router_groups=4), dict(router_top_groups=2),
               dict(router_groups=8, router_top_groups=1), dict(router_group_score="mean")):
        with pytest.raises(ValueError):
            M(128, 128, 16, 4, **kw)
    with pytest.raises(ValueError, match="format"):
        m.set_routed_weights(torch.zeros(16, 128, 256, dtype=BF16), torch.zeros(16, 128, 128, dtype=BF16), "int8")
    with pytest.raises(ValueError, match="shared"):
        M(128, 128, 16, 4, shared_expert=False).quantize_shared()


def test_fake_shapes_of_the_torch_operators():
    pkg()
    t, c, e, k, f = 10, 256, 8, 2, 128
    with FakeTensorMode():
        x = cuda(t, c)
        top, gate = torch.ops.praxis_b200.route_groups(cuda(t, e, dtype=torch.float32), None, k, "sigmoid", 4, 2, "max")
        assert (top.shape, top.dtype, gate.shape, gate.dtype) == ((t, k), torch.int64, (t, k), BF16)
        y = torch.ops.praxis_b200.fp8_linear(cuda(2, 5, c), *weight(300, c))
        assert (y.shape, y.dtype) == ((2, 5, 300), BF16)
        assert torch.ops.praxis_b200.fp8_mlp(x, *weight(2 * f, c), *weight(c, f)).shape == (t, c)
        y = torch.ops.praxis_b200.fp8_moe_forward(x, top, gate, *weight(e, 2 * f, c), *weight(e, c, f), 2.5, None)
        assert (y.shape, y.dtype) == ((t, c), BF16)


# -- kernels that overlap their predecessor --------------------------------------

CSRC = Path(pkg().build.__file__).parent / "csrc"


def code(name):
    """A source file without its comments."""
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def test_fp8_kernels_read_their_predecessors_results_with_ordinary_loads():
    """A kernel that is launched before the previous one has ended may read what
    that one writes with coherent loads only: read-only ones (__ldg, .nc, const
    __restrict__ parameters) are for weights and their scales."""
    fp8 = code("fp8.cu")
    assert set(re.findall(r"__ldg\(\s*(\w+)", fp8)) <= {"ws"}
    for name in ("common.cuh", "tail.cu", "fp8.cu"):
        assert "ld.global.nc" not in code(name)
    for kernel in ("fp8_slots_kernel", "fp8_quantize_kernel"):
        params = re.search(kernel + r"\(([^)]*)\)\s*\{", fp8).group(1)
        assert not re.search(r"const \w+\* __restrict__", params)


def test_grouped_router_reads_the_logits_with_ordinary_loads():
    """The logits kernel is its predecessor."""
    kernel = re.search(r"route_groups_kernel\(.*?\n}\n", code("router.cu"), re.S).group(0)
    assert "__ldg" not in kernel
    assert not re.search(r"const \w+\* __restrict__", kernel[: kernel.index("{")])


def test_the_streamed_tails_dispatch_is_complete_before_its_combine_starts():
    """The kernel right before the combine, which may still run when the combine
    starts, writes the rows alone."""
    ffn = code("capi.cu")
    ffn = ffn[ffn.index("int praxis_b200_fp8_ffn("):]
    assert ffn.index("run_fp8_identity(") < ffn.index("run_fp8_stream_ffn(") < ffn.index("run_combine_tail(")


def test_no_overlapping_kernel_reads_its_inputs_as_read_only_data():
    """The same for every kernel that waits for its predecessor, and for the device
    functions beside them."""
    for path in sorted(CSRC.glob("*.cu*")):
        text = code(path.name)
        if "pdl_wait" not in text and path.suffix == ".cu":
            continue
        for name, params, body in re.findall(r"\b(\w+)\(([^()]*)\)\s*\{(.*?)\n}\n", text, re.S):
            if name + "<<<" in text:
                continue  # launched behind its predecessor's end
            assert not re.search(r"const \w+\* __restrict__", params), (path.name, name)
            assert set(re.findall(r"__ldg\(\s*(\w+)", body)) <= {"ws"}, (path.name, name)


# -- workspaces --------------------------------------------------------------------

def ffn_workspace(tokens, top_k, experts, dim, hidden):
    p = pkg()
    p.build.build()
    return p.capi.load().praxis_b200_fp8_ffn_workspace_size(tokens, top_k, experts, dim, hidden)


@pytest.mark.parametrize("tokens", [1, 2, 6, 40, 1000])
def test_workspace_follows_the_routed_slots_and_not_the_experts(tokens):
    """At most min(E, slots) experts have rows, each padded by fewer than a tile."""
    c, f, e, k = 7168, 2048, 256, 8
    slots = tokens * k
    rows = (slots + 127 * min(e, slots)) // 128 * 128
    per_row = c + c // 128 * 4 + f + f // 128 * 4 + 2 * c  # codes and scales twice, the down rows in bf16
    size = ffn_workspace(tokens, k, e, c, f)
    assert size <= rows * per_row + slots * 8 + rows // 128 * 16 + 4 * (e + 1) * 3 + 32 * 4 * (c + f) // 128 + 4096
    if slots <= 8 + e // 8:  # streamed: fp32 hidden rows, and what a fused tail needs
        assert size <= slots * f * 4 + tokens * (c * 2 + 18) + 16 + 7 * 256


def test_workspace_of_no_tokens_is_empty():
    assert ffn_workspace(0, 8, 256, 7168, 2048) == 0
    assert ffn_workspace(0, 0, 1, 1024, 512) == 0
