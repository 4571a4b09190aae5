"""``llmop_fc_q4a``: the callable the reference's model builds for every
``nn.Linear`` (``chatllama/main.py:158-177``), and ``llmop_embedding_q8c``, the
one it builds for the token table (``chatllama/main.py:207-219``), on the GPU
kernels; and, with no counterpart in the reference, ``llmop_moe_q4a`` and
``llmop_fc_q4a_lora``, whose weights depend on the row."""
from __future__ import annotations

import torch

from . import llmops


class llmop_fc_q4a:
    """Packs ``linear.weight`` at construction, ``__call__(input)`` runs the FC
    and adds the bias.  Attributes as in the reference: ``weight`` (packed),
    ``bias``, ``N``.  ``qtype`` / ``group_k`` choose the block type that the
    reference fixes at compile time."""

    def __init__(self, linear, *, qtype="q4_1", group_k: int = 32, device=None) -> None:
        w = linear.weight.detach()
        dev = torch.device(device) if device is not None else (w.device if w.is_cuda else torch.device("cuda"))
        w = w.to(device=dev, dtype=torch.float32).contiguous()
        self.weight = llmops.offline_FC_quant_Q4A(w, qtype=qtype, group_k=group_k)
        b = getattr(linear, "bias", None)
        self.bias = b.detach().to(device=dev, dtype=torch.float32).contiguous() if b is not None else None
        self.N = int(linear.weight.shape[0])

    def __call__(self, input: torch.Tensor, **kw) -> torch.Tensor:
        if self.bias is not None and input.shape[0] * input.shape[1] <= 8 and kw.get("path", "auto") in ("auto", "decode"):
            # the reference's llmops.iadd(out, bias), folded into the decode kernel (same single fp32 add)
            return llmops.fc_Q4A(input, self.weight, self.N, addend=self.bias, **kw)
        out = llmops.fc_Q4A(input, self.weight, self.N, **kw)
        if self.bias is not None:
            out.add_(self.bias)  # the reference's llmops.iadd(out, bias)
        return out

    def weight_size(self) -> int:
        size = self.weight.numel() * self.weight.element_size()
        if self.bias is not None:
            size += self.bias.numel() * self.bias.element_size()
        return size

    def __repr__(self) -> str:
        return f"llmop_fc_q4a(weight: {list(self.weight.shape)})"


class llmop_embedding_q8c:
    """Quantizes the table at construction (one scale per row), ``__call__(input_ids)`` looks rows up and
    dequantizes them.  Attributes as in the reference: ``weight`` (int8 codes ``[V, E]``), ``scales`` (``[V]``)."""

    def __init__(self, weight: torch.Tensor, *, device=None) -> None:
        w = weight.detach()
        dev = torch.device(device) if device is not None else (w.device if w.is_cuda else torch.device("cuda"))
        self.weight, self.scales = llmops.embedding_q8c_quant_w(w.to(device=dev, dtype=torch.float32).contiguous())

    def __call__(self, input_ids: torch.Tensor) -> torch.Tensor:
        ids = input_ids.to(self.weight.device).contiguous()
        return llmops._front().embedding(ids, self.weight, self.scales, None)

    def __repr__(self) -> str:
        return f"llmop_embedding_q8c(weight: {list(self.weight.shape)})"


def _device_of(w: torch.Tensor, device) -> torch.device:
    return torch.device(device) if device is not None else (w.device if w.is_cuda else torch.device("cuda"))


class llmop_moe_q4a:
    """A layer of experts in place of one MLP (``chatllama/main.py:362-370`` per expert): the ``top_k`` experts that a
    router chose for a token, each ``down(silu(gate(x)) * up(x))``, summed with the router's weights.

    ``experts``: ``(gate, up, down)`` Linears without bias, all of the same sizes.  Gate and up are packed as one tensor, gate's
    columns first.  ``gate_up`` / ``down``: the packed tensors, ``[experts, Ng, Kg, block_bytes]``."""

    def __init__(self, experts, top_k: int, *, renormalize: bool = True, qtype="q4_1", group_k: int = 32, device=None) -> None:
        experts = list(experts)
        if not experts:
            raise RuntimeError("llmop_moe_q4a: no experts")
        sizes = {tuple(tuple(m.weight.shape) for m in e) for e in experts}
        inner, hidden = experts[0][0].weight.shape
        if sizes != {((inner, hidden), (inner, hidden), (hidden, inner))}:
            raise RuntimeError(f"llmop_moe_q4a: experts of sizes {sorted(sizes)}: expected gate and up [inner, hidden], down [hidden, inner]")
        if any(getattr(m, "bias", None) is not None for e in experts for m in e):
            raise RuntimeError("llmop_moe_q4a: experts have no bias")
        dev = _device_of(experts[0][0].weight, device)

        def packed(*parts):
            w = torch.cat([m.weight.detach().to(device=dev, dtype=torch.float32) for m in parts])
            return llmops.offline_FC_quant_Q4A(w.contiguous(), qtype=qtype, group_k=group_k)

        self.gate_up = torch.stack([packed(gate, up) for gate, up, _ in experts])
        self.down = torch.stack([packed(down) for _, _, down in experts])
        self.hidden, self.inner, self.top_k, self.renormalize = int(hidden), int(inner), int(top_k), renormalize

    def __call__(self, input: torch.Tensor, logits: torch.Tensor) -> torch.Tensor:
        """``input`` fp32 ``[B, M, hidden]``, ``logits`` fp32 ``[B, M, experts]`` (-inf: closed) -> ``[B, M, hidden]``."""
        if logits.shape[-1] != self.down.shape[0]:
            raise RuntimeError(f"llmop_moe_q4a: logits of {logits.shape[-1]} experts, there are {self.down.shape[0]}")
        weights, groups = llmops.route_top_k(logits, self.top_k, renormalize=self.renormalize)
        both = llmops.fc_Q4A_experts(input, self.gate_up, 2 * self.inner, groups)
        return llmops.fc_Q4A_experts(both, self.down, self.hidden, groups, weights=weights, silu_mul=True)

    def weight_size(self) -> int:
        return self.gate_up.numel() + self.down.numel()

    def __repr__(self) -> str:
        return f"llmop_moe_q4a(gate_up: {list(self.gate_up.shape)}, down: {list(self.down.shape)}, top_k: {self.top_k})"


class llmop_fc_q4a_lora(llmop_fc_q4a):
    """``llmop_fc_q4a`` with low-rank adapters beside it, one per row of the input.

    ``adapters``: ``(A, B, scale)`` each, ``A`` ``[rank, K]``, ``B`` ``[N, rank]``; lower ranks are filled up with zeros to the
    highest.  ``dtype``: what they are kept in (default: that of the first ``A``)."""

    def __init__(self, linear, adapters, *, dtype: torch.dtype | None = None, qtype="q4_1", group_k: int = 32, device=None) -> None:
        adapters = list(adapters)
        if not adapters:
            raise RuntimeError("llmop_fc_q4a_lora: no adapters")
        N, K = linear.weight.shape
        for a, b, _ in adapters:
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != K or b.shape[0] != N or a.shape[0] != b.shape[1]:
                raise RuntimeError(f"llmop_fc_q4a_lora: adapter {list(a.shape)}, {list(b.shape)} beside a weight {[N, K]}")
        super().__init__(linear, qtype=qtype, group_k=group_k, device=device)
        dev, rank = self.weight.device, max(a.shape[0] for a, _, _ in adapters)
        dtype = dtype or adapters[0][0].dtype
        self.lora_a = torch.zeros(len(adapters), rank, K, dtype=dtype, device=dev)
        self.lora_b = torch.zeros(len(adapters), N, rank, dtype=dtype, device=dev)
        for i, (a, b, _) in enumerate(adapters):
            self.lora_a[i, : a.shape[0]] = a.detach().to(device=dev, dtype=dtype)
            self.lora_b[i, :, : a.shape[0]] = b.detach().to(device=dev, dtype=dtype)
        self.scales = torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=dev)

    def __call__(self, input: torch.Tensor, groups: llmops.RowGroups, *, nibble_signed: bool = False) -> torch.Tensor:
        """``groups``: ``llmops.group_rows`` of the rows' adapters ``[B, M]`` (-1: none), made once for all Linears of a step."""
        out = llmops.fc_Q4A_lora(input, self.weight, self.N, self.lora_a, self.lora_b, groups, scales=self.scales,
                                 nibble_signed=nibble_signed)
        if self.bias is not None:
            out.add_(self.bias)  # the reference's llmops.iadd(out, bias)
        return out

    def weight_size(self) -> int:
        return super().weight_size() + sum(t.numel() * t.element_size() for t in (self.lora_a, self.lora_b, self.scales))

    def __repr__(self) -> str:
        return f"llmop_fc_q4a_lora(weight: {list(self.weight.shape)}, adapters: {list(self.lora_a.shape)})"
