"""Mixture-of-experts step on 8-bit integer weights.

``Int8ExpertBank`` holds all experts of a layer as int8 codes with a scale for each output channel;
``int8_moe_step`` is ``moe.moe_step`` over such a bank: router, experts, shared expert and ordered combine
on the device, activations quantised per token and, in front of the down projections, per (token,
expert).  ``moe_step`` hands a call with an ``Int8ExpertBank`` over to it, so ``ExpertsInference``,
``Qwen3NextMoEInference`` and ``ResidentExpertExecutor`` take such banks as they take packed ones.
"""
import ctypes
from functools import lru_cache

import torch

from . import _lib
from .int8_linear import Int8Weight, _call, _codes_of, _tiles_of, int8_quantize
from .quantized_linear import _TORCH_DTYPE_ID

_STEP_TOKENS = 4096       # tokens a call works on at a time: bounds the workspace of long prompts


@lru_cache(maxsize=4096)
def _workspace_bytes(*sizes):
    return _lib.load().qmoe_int8_moe_workspace_bytes(*sizes)


def _held(name):
    """A bank's tensor.  Another may take its place if it is what the kernels read there."""
    slot = "_" + name

    def put(self, tensor):
        old = getattr(self, slot)
        if not isinstance(tensor, torch.Tensor) or tensor.dtype != old.dtype or tensor.shape != old.shape or not tensor.is_contiguous():
            raise ValueError(f"{name} must be contiguous {str(old.dtype)[6:]} {list(old.shape)}")
        if tensor.device != old.device:
            raise ValueError("all matrices of a bank must be on the same device")
        setattr(self, slot, tensor)

    return property(lambda self: getattr(self, slot), put)


class Int8ExpertBank:
    """E SwiGLU experts: ``gate`` and ``up`` are (codes int8 [E, F, D], scales fp32 [E, F]) pairs, ``down`` is
    (codes int8 [E, D, F], scales fp32 [E, D]), contiguous on one device."""

    gate_tiles, up_tiles, down_tiles = _held("gate_tiles"), _held("up_tiles"), _held("down_tiles")
    gate_scales, up_scales, down_scales = _held("gate_scales"), _held("up_scales"), _held("down_scales")

    def __init__(self, gate, up, down):
        for name, pair in (("gate", gate), ("up", up), ("down", down)):
            if not isinstance(pair, (tuple, list)) or len(pair) != 2:
                raise TypeError(f"{name} must be a (codes, scales) pair")
        if gate[0].shape != up[0].shape:
            raise ValueError("gate/up banks must share [E, F, D]")
        if gate[0].ndim != 3:
            raise ValueError("expert banks are three-dimensional [E, N, K]")
        e, f, d = (int(i) for i in gate[0].shape)
        if tuple(down[0].shape) != (e, d, f):
            raise ValueError("down bank must be [E, D, F]")
        if not gate[0].device == up[0].device == down[0].device:
            raise ValueError("all matrices of a bank must be on the same device")
        self._hold(tuple(_tiles_of(codes, scales, 3, "Int8 expert bank") for codes, scales in (gate, up, down)),
                   (gate[1], up[1], down[1]), e, d, f)

    def _hold(self, tiles, scales, e, d, f):
        self._gate_tiles, self._up_tiles, self._down_tiles = tiles
        self._gate_scales, self._up_scales, self._down_scales = scales
        self._sizes = tuple(t.numel() for t in (*tiles, *scales))
        self.n_experts, self.d_model, self.d_ff = e, d, f
        self.device = tiles[0].device

    def fill(self, args):
        """The bank's part of a step's argument struct.  Addresses are read from the tensors at every call: one kept from an
        earlier call would be stale, or free, once a tensor is replaced."""
        gate, up, down, gs, us, ds = (self._gate_tiles, self._up_tiles, self._down_tiles, self._gate_scales, self._up_scales, self._down_scales)
        if (gate.numel(), up.numel(), down.numel(), gs.numel(), us.numel(), ds.numel()) != self._sizes:
            raise ValueError("a tensor of the bank was resized")
        args.gate, args.up, args.down = gate.data_ptr(), up.data_ptr(), down.data_ptr()
        args.gate_scales, args.up_scales, args.down_scales = gs.data_ptr(), us.data_ptr(), ds.data_ptr()
        args.n_experts, args.d_model, args.d_ff = self.n_experts, self.d_model, self.d_ff

    @classmethod
    def from_packed(cls, bank):
        """From a ``DevicePackedExpertBank``: every expert's dequantised rows, quantised (expert by expert, so
        only one dense expert exists at a time)."""
        from .moe import DevicePackedExpertBank
        if not isinstance(bank, DevicePackedExpertBank):
            raise TypeError("Expected DevicePackedExpertBank")
        lib = _lib.load()
        e, d, f = bank.n_experts, bank.d_model, bank.d_ff
        shapes = ((f, d), (f, d), (d, f))
        sizes = [lib.qmoe_int8_matrix_bytes(n, k) for n, k in shapes]
        tiles = tuple(torch.empty(e * size, dtype=torch.uint8, device=bank.device) for size in sizes)
        scales = tuple(torch.empty((e, n), dtype=torch.float32, device=bank.device) for n, _ in shapes)
        for i in range(e):
            for at, packed in enumerate(bank.expert(i)):
                codes, s = int8_quantize(packed.dequantize())
                tiles[at][i * sizes[at]:(i + 1) * sizes[at]] = _tiles_of(codes, s, 2, "Int8 expert bank")
                scales[at][i] = s
        self = cls.__new__(cls)
        self._hold(tiles, scales, e, d, f)
        return self

    @property
    def nbytes(self):
        return sum(int(t.numel()) for t in (self.gate_tiles, self.up_tiles, self.down_tiles)) + 4 * sum(
            int(s.numel()) for s in (self.gate_scales, self.up_scales, self.down_scales))

    @property
    def expert_nbytes(self):
        return self.nbytes // self.n_experts

    def expert(self, index):
        """One expert as three ``Int8Weight`` matrices (the tiles are views, nothing is copied)."""
        i = int(index)
        if not 0 <= i < self.n_experts:
            raise IndexError(index)
        out = []
        for tiles, scales, shape in ((self.gate_tiles, self.gate_scales, (self.d_ff, self.d_model)),
                                     (self.up_tiles, self.up_scales, (self.d_ff, self.d_model)),
                                     (self.down_tiles, self.down_scales, (self.d_model, self.d_ff))):
            size = tiles.numel() // self.n_experts
            w = Int8Weight.__new__(Int8Weight)
            w.tiles, w.scales, w.shape, w.device = tiles[i * size:(i + 1) * size], scales[i], shape, self.device
            out.append(w)
        return tuple(out)

    def codes(self, index):
        """The row-major int8 codes (gate, up, down) of one expert."""
        return tuple(_codes_of(w.tiles, w.shape) for w in self.expert(index))


def _given(tensor, dtype, shape, device, what):
    """Address of an operand after its checks."""
    if not isinstance(tensor, torch.Tensor) or tensor.dtype != dtype or tensor.shape != shape or not tensor.is_contiguous():
        raise ValueError(f"{what} must be contiguous {str(dtype)[6:]} {list(shape)}")
    if tensor.device != device:
        raise ValueError("all operands must be on the same device")
    return tensor.data_ptr()


def int8_moe_step(hidden, bank, top_k, *, logits=None, weights=None, ids=None, shared=None, shared_gate=None, floor=2.0 ** -14,
                  renormalize=True, out_dtype=None, return_routing=False, residual=None, check_routing=False):
    """One MoE step over ``hidden`` [T, D] with an ``Int8ExpertBank``: routed experts (+ shared expert) -> [T, D].

    The arguments are those of ``moe.moe_step``; ``shared`` is an optional (gate, up, down) triple of
    ``Int8Weight``.  A token's experts are added in ascending id, each weighted output rounded to fp32 before
    it is added, and the sum is rounded once to ``out_dtype`` (default: hidden's type).  A token whose hidden
    row is not finite gets NaN; the other tokens are not touched by it.
    """
    if not isinstance(bank, Int8ExpertBank):
        raise TypeError("Expected Int8ExpertBank")
    if not isinstance(hidden, torch.Tensor) or not hidden.is_cuda or hidden.dtype not in _TORCH_DTYPE_ID:
        raise TypeError("MoE hidden must be a CUDA FP16/BF16/FP32 tensor")
    e, d, f, device = bank.n_experts, bank.d_model, bank.d_ff, bank.device
    if hidden.ndim != 2 or hidden.shape[1] != d or not hidden.is_contiguous():
        raise ValueError("hidden must be contiguous [tokens, d_model]")
    if hidden.device != device:
        raise ValueError("all operands must be on the same device")
    out_dtype = hidden.dtype if out_dtype is None else out_dtype
    if out_dtype not in _TORCH_DTYPE_ID:
        raise TypeError("out_dtype must be FP16, BF16, or FP32")
    t, k = hidden.shape[0], int(top_k)
    if not 1 <= k <= min(32, e) or e > 4096:
        raise NotImplementedError("the step covers at most 4096 experts and 1 <= top_k <= min(32, experts)")
    args = _lib.Int8MoeArgs()
    bank.fill(args)
    lg = iw = ii = rs = None
    if logits is not None:
        lg = _given(logits, torch.float32, (t, e), device, "router logits")
    elif weights is None or ids is None:
        raise ValueError("need router logits or weights and ids")
    else:
        iw = _given(weights, torch.float32, (t, k), device, "routing weights")
        ii = _given(ids, torch.int64, (t, k), device, "routing ids")
    if residual is not None:
        rs = _given(residual, torch.float32, (t, d), device, "residual")
    fs = 0
    if shared is not None:
        if len(shared) != 3 or not all(isinstance(w, Int8Weight) for w in shared):
            raise TypeError("shared expert: a (gate, up, down) triple of Int8Weight")
        g, u, dn = shared
        fs = g.shape[0]
        if g.shape != (fs, d) or u.shape != (fs, d) or dn.shape != (d, fs):
            raise ValueError("shared expert must be [Fs, D], [Fs, D], [D, Fs]")
        if not g.device == u.device == dn.device == device:
            raise ValueError("all operands must be on the same device")
        args.shared_gate_w, args.shared_up_w, args.shared_down_w = g.tiles.data_ptr(), u.tiles.data_ptr(), dn.tiles.data_ptr()
        args.shared_gate_scales, args.shared_up_scales, args.shared_down_scales = (
            g.scales.data_ptr(), u.scales.data_ptr(), dn.scales.data_ptr())
        args.d_ff_shared = fs
        if shared_gate is not None:
            args.shared_gate = _given(shared_gate, torch.float32, (d,), device, "shared_gate")
    out = hidden.new_empty((t, d), dtype=out_dtype)
    out_w = hidden.new_empty((t, k), dtype=torch.float32) if return_routing else None
    out_i = hidden.new_empty((t, k), dtype=torch.int64) if return_routing else None
    if t == 0:
        return (out, out_w, out_i) if return_routing else out
    step = min(t, _STEP_TOKENS)
    nbytes = _workspace_bytes(step, k, e, d, f, fs)
    workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
    status = torch.zeros(1, dtype=torch.int32, device=device) if check_routing else None
    args.hidden_dtype, args.out_dtype, args.top_k = _TORCH_DTYPE_ID[hidden.dtype], _TORCH_DTYPE_ID[out_dtype], k
    args.floor_value, args.renormalize = float(floor), int(bool(renormalize))
    if status is not None:
        args.status_out = status.data_ptr()
    function = _lib.load().qmoe_int8_moe_forward
    for lo in range(0, t, step):
        args.tokens = min(step, t - lo)
        args.hidden, args.out = hidden.data_ptr() + lo * d * hidden.element_size(), out.data_ptr() + lo * d * out.element_size()
        if lg is not None:
            args.logits = lg + lo * e * 4
        else:
            args.in_weights, args.in_ids = iw + lo * k * 4, ii + lo * k * 8
        if rs is not None:
            args.residual = rs + lo * d * 4
        if return_routing:
            args.out_weights, args.out_ids = out_w.data_ptr() + lo * k * 4, out_i.data_ptr() + lo * k * 8
        rc = _call(device, function, ctypes.byref(args), workspace.data_ptr(), nbytes)
        if rc:
            _lib.check(rc, "Int8 MoE step")
    if status is not None:
        bits = int(status.item())
        if bits:
            what = [name for bit, name in ((1, "expert ids outside the bank"), (2, "an expert repeated within a token")) if bits & bit]
            raise ValueError("Invalid routing: " + " and ".join(what))
    return (out, out_w, out_i) if return_routing else out
