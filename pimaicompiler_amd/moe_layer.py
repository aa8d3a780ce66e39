"""A mixture-of-experts layer for a few tokens: router, choice, the chosen experts' products and their weighted sum.

MoePlan (ops.py) is the step for one token and one expert in fp16 in a single launch; this is the layer of a served model: any number of
experts per token, fp16 or bf16, gated or not, weights in 16 or 4 bits, a batch of tokens at a time."""
import ctypes
import weakref

import torch

from . import _lib as L
from .mx4 import _CODES, Mx4Tensor, _require, _rows_of
from .ops import NNRuntimeException, _check, _ensure_init, _Launch, _native, _require_no_gradient, _result

TOKENS_MOST = 64  # tokens of one launch; longer inputs are taken in pieces of that many
_ACTS = {"none": L.PIMHIP_EXPERT_NONE, "aten::relu": L.PIMHIP_EXPERT_RELU, "aten::silu": L.PIMHIP_EXPERT_SILU}


class MoeLayerPlan:
    """y = sum over a token's top_k experts of share * (W2 act(W1 x + b1) + b2).

    router = (W_r [E, d_model], b_r [E] or None); w1[e] [d_ff, d_model] and w2[e] [d_model, d_ff], as lists or as stacked tensors, in the
    router's type (fp16 or bf16), or lists of Mx4Tensor; b1[e] [d_ff] and b2[e] [d_model] or None.  gated: w1[e] is [2 d_ff, d_model]
    (and b1[e] [2 d_ff]), the gate's rows first, and hidden = act(gate) * value.  act_type "none", "aten::relu" or "aten::silu".
    renormalize: a token's shares are the softmax over its chosen experts; else over all.

    Sums and hidden values are fp32, so y is rounded once.  E up to 256, top_k up to 16, d_model a multiple of 8.  The plan reads the weights where they lie (contiguous copies where they are
    not contiguous) and may be used on several streams at a time."""

    def __init__(self, router, w1, w2, b1=None, b2=None, top_k=2, act_type="aten::silu", gated=False, renormalize=True, stream=None):
        wr, br = router
        _require("router weight", wr, (torch.float16, torch.bfloat16))
        E = len(w1)
        if wr.dim() != 2 or wr.size(0) != E or E < 1 or len(w2) != E or (b1 is not None and len(b1) != E) or (b2 is not None and len(b2) != E):
            raise NNRuntimeException("the router must be [E, d_model] with E experts in w1, w2 (and b1, b2)")
        if act_type not in _ACTS:
            raise NNRuntimeException(f"act_type={act_type!r} is none of {', '.join(_ACTS)}")
        w1, w2 = list(w1), list(w2)
        b1, b2 = (list(b) if b is not None else None for b in (b1, b2))
        mx4 = isinstance(w1[0], Mx4Tensor)
        self.d_model, self.num_experts, self.top_k, self.dtype, self.device = wr.size(1), E, int(top_k), wr.dtype, wr.device
        rows1 = w1[0].shape[0]
        if gated and rows1 % 2:
            raise NNRuntimeException("a gated layer's w1 holds as many gate rows as value rows")
        self.d_ff = rows1 // 2 if gated else rows1
        for e in range(E):
            for name, w, shape in (("w1", w1[e], (rows1, self.d_model)), ("w2", w2[e], (self.d_model, self.d_ff))):
                if isinstance(w, Mx4Tensor) != mx4:
                    raise NNRuntimeException("all experts' weights are Mx4Tensors or none")
                if not mx4:
                    _require(f"{name}[{e}]", w, (self.dtype,))
                if tuple(w.shape) != shape or w.device != self.device:
                    raise NNRuntimeException(f"{name}[{e}] must be {list(shape)} on {self.device}, got {list(w.shape)} on {w.device}")
        for name, bs, n in (("router bias", [br] if br is not None else [], E), ("b1", b1 or [], rows1), ("b2", b2 or [], self.d_model)):
            for b in bs:
                _require(name, b, (self.dtype,))
                if b.numel() != n or b.device != self.device:
                    raise NNRuntimeException(f"{name} must have {n} elements on {self.device}")
        if not mx4:
            _require_no_gradient(*w1, *w2)
        _require_no_gradient(wr, br, *(b1 or []), *(b2 or []))
        _ensure_init(wr)
        with _Launch(self.device, stream) as handle:
            keep = []

            def at(t):
                keep.append(t.contiguous())
                if keep[-1].data_ptr() % 16:   # (a weight at an odd offset of a larger tensor)
                    keep[-1] = keep[-1].clone()
                return keep[-1].data_ptr()

            def table(ts):
                return (ctypes.c_void_p * E)(*[at(t) for t in ts]) if ts is not None else None
            d = L.MoeLayerDesc()
            d.router_w, d.router_b = at(wr), at(br) if br is not None else None
            if mx4:
                keep += w1 + w2
                d.w1_mx4, d.w2_mx4 = (L.Mx4Matrix * E)(*[w._c for w in w1]), (L.Mx4Matrix * E)(*[w._c for w in w2])
            else:
                d.w1, d.w2 = table(w1), table(w2)
            d.b1, d.b2 = table(b1), table(b2)
            d.d_model, d.d_ff, d.num_experts, d.top_k = self.d_model, self.d_ff, E, self.top_k
            d.dtype, d.act, d.gated, d.renormalize = _CODES[self.dtype], _ACTS[act_type], int(bool(gated)), int(bool(renormalize))
            plan = ctypes.c_void_p()
            _check(L.load().pimhip_moe_layer_plan_create(ctypes.byref(plan), ctypes.byref(d), handle))
        self._keep = keep
        self._handle = plan
        self._finalizer = weakref.finalize(self, MoeLayerPlan._destroy, plan.value)

    @staticmethod
    def _destroy(handle_value):
        try:
            L.load().pimhip_moe_layer_plan_destroy(ctypes.c_void_p(handle_value))
        except Exception:  # interpreter shutdown
            pass

    def workspace_bytes(self, tokens):
        """What a call with that many tokens needs besides its outputs."""
        n = ctypes.c_uint64()
        _check(L.load().pimhip_moe_layer_workspace_bytes(self._handle, tokens, ctypes.byref(n)))
        return n.value

    def forward(self, x, stream=None):
        """y [.., d_model], experts [.., top_k] int32, shares [.., top_k] fp32 for x [.., d_model]: the experts in falling order of their logits,
        equal ones by their index.  Nothing is read back.  More than 64 tokens are taken 64 at a time."""
        out = _native().fast_moe_layer(self._handle.value, x, self.d_model, self.top_k, _CODES[self.dtype], self.device.index, TOKENS_MOST) if stream is None else None
        if out is not None:
            return _result(out)
        _require("x", x, (self.dtype,))
        _require_no_gradient(x)
        if x.dim() < 1 or x.size(-1) != self.d_model or x.device != self.device:
            raise NNRuntimeException(f"x must be [.., {self.d_model}] on {self.device}, got {tuple(x.shape)} on {x.device}")
        lib = L.load()
        with _Launch(self.device, stream, x) as handle:
            x2, ld = _rows_of(x)
            M, k = x2.size(0), self.top_k
            y = torch.empty(x.shape, dtype=self.dtype, device=self.device)
            experts = torch.empty((*x.shape[:-1], k), dtype=torch.int32, device=self.device)
            shares = torch.empty((*x.shape[:-1], k), dtype=torch.float32, device=self.device)
            workspace = torch.empty(self.workspace_bytes(min(M, TOKENS_MOST)), dtype=torch.uint8, device=self.device)
            for first in range(0, M, TOKENS_MOST):
                n = min(TOKENS_MOST, M - first)
                _check(lib.pimhip_moe_layer_forward(self._handle, x2.data_ptr() + first * ld * 2, ld, n, y.data_ptr() + first * self.d_model * 2,
                                                    experts.data_ptr() + first * k * 4, shares.data_ptr() + first * k * 4, workspace.data_ptr(), handle))
        return y, experts, shares
