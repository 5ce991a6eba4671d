"""Low-rank adapters of many requests beside a shared projection, on the GPU: forward and gradients.

    out[m] = act(y[m] + scaling[a] (x[m] down[a]^T) up[a]^T),  a = ids[m]

A 4-bit weight cannot be tuned itself; the adapters are what is trained and swapped, per request, while all requests of a batch
share the projection (`LinearGQ.build(x, adapters=, plan=)`, `LinearGQ.grad`).
"""
import ctypes

from popxl_addons import _gq_hip

__all__ = ["AdapterPlan", "LowRankAdapters", "low_rank_adapters", "low_rank_adapters_grad"]


class LowRankAdapters:
    """The adapters of one projection: down float16 [n_adapters, rank, in_features], up float16 [n_adapters, out_features, rank]
    (each adapter's matrices as they are published: y += scaling * up @ (down @ x)), scaling float32 [n_adapters] or one number.
    rank is at most 128, n_adapters at most 2048.  Adapters of lower rank are padded with zeros.  The tensors are kept, not
    copied: writing to them changes the adapters."""

    def __init__(self, down, up, scaling=1.0):
        import torch

        if down.dim() != 3 or up.dim() != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2]:
            raise ValueError("LowRankAdapters: down must be [n_adapters, rank, in] and up [n_adapters, out, rank], got "
                             f"{tuple(down.shape)} and {tuple(up.shape)}")
        if down.dtype != torch.float16 or up.dtype != torch.float16:
            raise TypeError("LowRankAdapters: down and up must be float16")
        if not 1 <= down.shape[1] <= 128 or not 1 <= down.shape[0] <= 2048:
            raise ValueError(f"LowRankAdapters: rank {down.shape[1]} outside 1 ... 128 or {down.shape[0]} adapters outside 1 ... 2048")
        if not isinstance(scaling, torch.Tensor):
            scaling = torch.full((down.shape[0],), float(scaling), dtype=torch.float32, device=down.device)
        if tuple(scaling.shape) != (down.shape[0],) or scaling.dtype != torch.float32:
            raise ValueError(f"LowRankAdapters: scaling must be float32 [{down.shape[0]}]")
        for t in (down, up, scaling):
            if not t.is_contiguous() or t.device != down.device:
                raise ValueError("LowRankAdapters: the tensors must be contiguous and on one device")
        self.down, self.up, self.scaling = down, up, scaling
        self.n_adapters, self.rank, self.in_features = down.shape
        self.out_features = up.shape[1]
        self.device, self.index = down.device, down.get_device()
        self._workspaces = {}  # bytes that a call needs, by entry point and rows
        self._c = _gq_hip.Adapters(down.data_ptr(), up.data_ptr(), scaling.data_ptr(), self.n_adapters, self.rank, self.in_features,
                                   self.out_features)

    def workspace(self, function, rows):
        """A new workspace for a call over `rows` rows (one that the allocator orders with the stream it is used on)."""
        import torch

        need = self._workspaces.get((function, rows))
        if need is None:
            need = getattr(_gq_hip.load(), function)(ctypes.byref(self._c), rows)
            if need < 0:
                raise _gq_hip.GQHipError(function, need, _gq_hip.last_error())
            if len(self._workspaces) > 256:
                self._workspaces.clear()
            self._workspaces[function, rows] = need
        return torch.empty(need, dtype=torch.uint8, device=self.device), need


class AdapterPlan:
    """The rows of a batch sorted by adapter, made once on the device and used for every projection that the batch passes.
    ids: int32 [rows], an adapter's number or anything outside [0, n_adapters) for a row without one."""

    def __init__(self, ids, n_adapters):
        import torch

        if not ids.is_cuda:
            raise RuntimeError("AdapterPlan runs on the GPU only: move ids to a HIP device")
        if not 1 <= n_adapters <= 2048:
            raise ValueError(f"AdapterPlan: {n_adapters} adapters outside 1 ... 2048")
        if ids.dim() != 1:
            raise ValueError(f"AdapterPlan: ids must be [rows], got {tuple(ids.shape)}")
        self.rows, self.n_adapters, self.device, self.index = ids.shape[0], n_adapters, ids.device, ids.get_device()
        nbytes = _gq_hip.load().gq_adapter_plan_bytes(self.rows, n_adapters)
        if nbytes < 0:
            raise _gq_hip.GQHipError("gq_adapter_plan_bytes", nbytes, _gq_hip.last_error())
        self.data = torch.empty(nbytes, dtype=torch.uint8, device=ids.device)
        self.update(ids)

    def update(self, ids):
        """Plan other ids of as many rows in the same memory (graphs captured with this plan then use them)."""
        import torch

        if ids.dtype != torch.int32:
            raise TypeError(f"AdapterPlan: ids must be int32, got {ids.dtype}")
        if ids.dim() != 1 or ids.shape[0] != self.rows or ids.get_device() != self.index:
            raise ValueError(f"AdapterPlan: ids must be [{self.rows}] on {self.device}")
        ids = ids.contiguous()
        _gq_hip.launch(self.index, "gq_adapter_plan", ids.data_ptr(), self.rows, self.n_adapters, self.data.data_ptr(), self.data.numel())


def _matrix(name, t, features, adapters, rows):
    """t [..., features] as float16 rows a stride apart."""
    import torch

    if not t.is_cuda:
        raise RuntimeError("low-rank adapters run on the GPU only: move the tensors to a HIP device")
    if t.dtype != torch.float16:
        raise TypeError(f"{name} must be float16, got {t.dtype}")
    if t.shape[-1] != features:
        raise ValueError(f"{name} must have {features} features, got {t.shape[-1]}")
    if t.get_device() != adapters.index:
        raise ValueError(f"{name} must be on the adapters' device")
    if t.dim() != 2 or t.stride(1) != 1:
        t = t.reshape(-1, features).contiguous()
    if t.shape[0] != rows:
        raise ValueError(f"{name} has {t.shape[0]} rows, the plan {rows}")
    return t


def _check_plan(adapters, plan):
    if plan.n_adapters != adapters.n_adapters or plan.index != adapters.index:
        raise ValueError(f"the plan is for {plan.n_adapters} adapters on {plan.device}, these are {adapters.n_adapters} on {adapters.device}")


def low_rank_adapters(x, y, adapters, plan, activation=None, out=None):
    """
    act(y + scaling (x down^T) up^T), each row with its adapter; rows without one: act(y).

    Args:
        x (torch.Tensor): float16 [..., in_features], what the shared projection read
        y (torch.Tensor): float16 [..., out_features], its result without an activation; None for zeros
        adapters (LowRankAdapters)
        plan (AdapterPlan): of the batch's rows
        activation: None, "relu", "gelu_tanh", applied behind the sum
        out (torch.Tensor): float16, 2-D with a contiguous last axis or contiguous; may be y; a new tensor if None

    Returns:
        torch.Tensor: `out`.  One rounding to float16; the intermediate product is kept in 32 bits.
    """
    import torch

    act, rows, features = _gq_hip.activation_code(activation), plan.rows, adapters.out_features
    _check_plan(adapters, plan)
    x2 = _matrix("x", x, adapters.in_features, adapters, rows)
    y2 = None if y is None else _matrix("y", y, features, adapters, rows)
    if out is None:
        out = x.new_empty((*x.shape[:-1], features))
    elif out.dtype != torch.float16 or out.shape[-1] != features or out.get_device() != adapters.index:
        raise ValueError(f"out must be float16 [..., {features}] on the adapters' device")
    out2 = out if out.dim() == 2 and out.stride(1) == 1 else out.view(-1, features)
    if out2.shape[0] != rows:
        raise ValueError(f"out has {out2.shape[0]} rows, the plan {rows}")
    workspace, nbytes = adapters.workspace("gq_adapter_apply_workspace_bytes", rows)
    _gq_hip.launch(adapters.index, "gq_adapter_apply_f16", ctypes.byref(adapters._c), plan.data.data_ptr(), rows, x2.data_ptr(), x2.stride(0),
                   0 if y2 is None else y2.data_ptr(), 0 if y2 is None else y2.stride(0), out2.data_ptr(), out2.stride(0), act,
                   workspace.data_ptr(), nbytes)
    return out


def low_rank_adapters_grad(x, dy, adapters, plan, dx=None):
    """
    Gradients of `low_rank_adapters` (without an activation) for dy = dL/dout.

    Args:
        x, dy (torch.Tensor): float16 [..., in_features] and [..., out_features]
        dx (torch.Tensor): float16 [..., in_features], the gradient that reaches x through the shared projection; None for zeros

    Returns:
        (dx + scaling dy up down, float16; d_down, float32 [n_adapters, rank, in]; d_up, float32 [n_adapters, out, rank]).
        Adapters without rows get zeros.  Sums are float32 in a fixed order: equal calls give equal bits.  (The gradient of y is dy.)
    """
    import torch

    _check_plan(adapters, plan)
    x2 = _matrix("x", x, adapters.in_features, adapters, plan.rows)
    dy2 = _matrix("dy", dy, adapters.out_features, adapters, plan.rows)
    dx2 = None if dx is None else _matrix("dx", dx, adapters.in_features, adapters, plan.rows)
    out = x.new_empty(x.shape)
    if plan.rows == 0 or adapters.in_features == 0 or adapters.out_features == 0:
        d_down, d_up = (torch.zeros(w.shape, dtype=torch.float32, device=w.device) for w in (adapters.down, adapters.up))
        return out.zero_() if dx is None else out.copy_(dx), d_down, d_up
    d_down, d_up = (torch.empty(w.shape, dtype=torch.float32, device=w.device) for w in (adapters.down, adapters.up))
    workspace, nbytes = adapters.workspace("gq_adapter_grad_workspace_bytes", plan.rows)
    _gq_hip.launch(adapters.index, "gq_adapter_grad_f16", ctypes.byref(adapters._c), plan.data.data_ptr(), plan.rows, x2.data_ptr(),
                   x2.stride(0), dy2.data_ptr(), dy2.stride(0), 0 if dx2 is None else dx2.data_ptr(), 0 if dx2 is None else dx2.stride(0),
                   out.data_ptr(), adapters.in_features, d_down.data_ptr(), d_up.data_ptr(), workspace.data_ptr(), nbytes)
    return out, d_down, d_up
