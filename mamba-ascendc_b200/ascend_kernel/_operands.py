"""Checks of arguments that the operators around a selective state space layer share: what a call says that ``_calls``
(csrc/torch_calls.cpp, which checks the same) did not take.

They raise ``RuntimeError("<operator>: ...")`` before any launch, as ``mamba2_ssd_fwd`` does
(mamba_ascendc/csrc/ops/mamba2_ssd_fwd/op_host/mamba2_ssd_fwd.cpp:15-112)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def fail(op: str, text: str) -> None:
    raise RuntimeError(f"{op}: {text}")


def unsupported(op: str) -> None:
    """The arguments are as they should be, but a tensor is not a plain one (its storage, layout or device)."""
    fail(op, "takes plain strided CUDA tensors only")


def underived(op: str, *tensors: Optional[torch.Tensor]) -> None:
    """Neither inside a function transform nor with forward-mode derivatives, which the kernels would lose."""
    tensors = [t for t in tensors if t is not None]
    transforms, forward = torch._C._functorch, torch.autograd.forward_ad
    if any(transforms.is_legacy_batchedtensor(t) or transforms.is_functorch_wrapped_tensor(t) for t in tensors):
        fail(op, "cannot run inside a function transform (vmap, grad, jvp)")
    if forward._current_level >= 0 and any(forward.unpack_dual(t).tangent is not None for t in tensors):
        fail(op, "has no forward-mode derivatives")


def activation(op: str, t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> None:
    """A CUDA tensor of one of the activations' types, its columns side by side; ``like`` says which type and device."""
    if not t.is_cuda:
        fail(op, f"{name} must be a CUDA tensor")
    if like is None:
        if t.dtype not in DTYPES:
            fail(op, f"{name} must be float32, bfloat16 or float16")
    elif t.dtype is not like.dtype:
        fail(op, f"{name} must have the type of x")
    elif t.device != like.device:
        fail(op, f"{name} must be on the device of x")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        fail(op, f"{name} must be contiguous in its last dimension")


def parameter(op: str, t: torch.Tensor, name: str, shape: Tuple[int, ...], like: torch.Tensor, f32_only: bool = False) -> None:
    """A contiguous tensor of ``shape`` in fp32 or, unless ``f32_only``, the type of x."""
    if t.dtype is not torch.float32 and (f32_only or t.dtype is not like.dtype):
        fail(op, f"{name} must be float32" + ("" if f32_only else " or have the type of x"))
    exactly(op, t, name, shape, like)


def exactly(op: str, t: torch.Tensor, name: str, shape: Tuple[int, ...], like: torch.Tensor) -> None:
    if t.device != like.device:
        fail(op, f"{name} must be on the device of x")
    if tuple(t.shape) != shape:
        fail(op, f"{name} must have shape {list(shape)}")
    if not t.is_contiguous():
        fail(op, f"{name} must be contiguous")


def packing(op: str, cu_seqlens: torch.Tensor, x: torch.Tensor) -> int:
    """Number of sequences packed in x [1, tokens, ...]."""
    if cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or not cu_seqlens.is_contiguous():
        fail(op, "cu_seqlens must be a contiguous int32 tensor [sequences + 1]")
    if cu_seqlens.device != x.device:
        fail(op, "cu_seqlens must be on the device of x")
    if x.shape[0] != 1:
        fail(op, "with cu_seqlens the batch must be 1")
    return cu_seqlens.numel() - 1


def slot_numbers(op: str, slots: Optional[torch.Tensor], x: torch.Tensor, state: torch.Tensor) -> None:
    """Which slot of a cache each row of x takes."""
    if slots is None:
        if state.shape[0] != x.shape[0]:
            fail(op, "without slots the state must have a row for each row of x")
        return
    if slots.dtype is not torch.int32 or tuple(slots.shape) != (x.shape[0],) or not slots.is_contiguous():
        fail(op, "slots must be a contiguous int32 tensor with a number for each row of x")
    if slots.device != x.device:
        fail(op, "slots must be on the device of x")


def cache(op: str, state: torch.Tensor, name: str, inner: Tuple[int, ...], dtype: torch.dtype, x: torch.Tensor) -> None:
    """[slots, *inner], each slot contiguous; slots may lie apart (one layer's share of a larger cache)."""
    if state.device != x.device:
        fail(op, f"{name} must be on the device of x")
    if state.dtype is not dtype:
        fail(op, f"{name} must be {str(dtype)[6:]}")
    if state.dim() != len(inner) + 1 or tuple(state.shape[1:]) != inner:
        fail(op, f"{name} must have shape [slots, {', '.join(map(str, inner))}]")
    want = 1
    for size, stride in zip(reversed(state.shape[1:]), reversed(state.stride()[1:])):
        if size > 1 and stride != want:
            fail(op, f"{name} must be contiguous within a slot")
        want *= size
    if state.shape[0] > 1 and state.stride(0) < want:
        fail(op, f"{name} must have its slots apart")


def apart(op: str, state: torch.Tensor, state_out: torch.Tensor) -> None:
    """Slot i of state_out may be slot i of state, and shares no memory with any other."""
    count, size = state.shape[0], state.element_size()
    inner = state[0].numel() * size if count else 0
    if inner == 0:
        return
    step, step_out = (t.stride(0) * size if count > 1 else inner for t in (state, state_out))
    distance = state_out.data_ptr() - state.data_ptr()
    if distance >= (count - 1) * step + inner or -distance >= (count - 1) * step_out + inner:
        return
    for i in range(count):
        at = distance + i * step_out
        k = max(at, 0) // step
        for near in range(k, min(k + 2, count)):
            if at < near * step + inner and near * step < at + inner and not (near == i and at == i * step):
                fail(op, "state_out must be state or lie apart from it")


def without_gradients(op: str, *tensors: Optional[torch.Tensor]) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        fail(op, "has no gradients; call it under torch.no_grad()")
