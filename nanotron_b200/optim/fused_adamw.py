"""AdamW over fp32 parameters (state-dict compatible with ``torch.optim.AdamW``).

On CUDA, when every parameter is a slice of ONE contiguous fp32 master buffer (what the fp32 gradient accumulator
builds) and its gradient / half-precision twin sit at a constant offset in their own flat buffers, the whole
optimizer step is a single launch of the in-tree flat kernel: gradient scaling (clipping coefficient read on the
device), AdamW, and the bf16 write-back of the updated weights, replacing the separate fp32->bf16 pass of the
reference (reference src/nanotron/optim/gradient_accumulator.py:255-267).  The ``exp_avg`` / ``exp_avg_sq`` states
are views of two flat buffers with the same layout.  Scattered tensors take one launch of the multi-tensor kernel
(``ops.adamw_multi_tensor``); what that has no form for (fp16, strided parameters, bf16 states) runs per tensor.

``state_bits=8`` keeps both averages as 8-bit codes with one exponent byte per 128 elements: 2.02 bytes per parameter instead
of 8.  The state dict holds them as fp32 tensors all the same (an 8-bit value is exact there, and encoding it again gives the
same codes), so checkpoints move freely between both forms and between layouts.
"""
from __future__ import annotations

from typing import Dict, List, Optional

import torch

from nanotron_b200.ops import reference as ref


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits: int = 32, state_seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 8 or 32, got {state_bits}")
        self.state_bits = state_bits
        self.state_seed = state_seed  # of the stochastic rounding of 8-bit states; mixed with the step number
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)
        self.half_targets: Dict[int, torch.Tensor] = {}  # id(master) -> flat half-precision destination view
        self.grad_scale: Optional[torch.Tensor] = None  # optional device scalar multiplied into every gradient
        self._flat = None  # cached flat plan
        self._flat_failed = False

    def set_half_target(self, master: torch.Tensor, half_view: torch.Tensor):
        """After each step also write ``master`` (cast) into ``half_view`` (same numel)."""
        assert master.numel() == half_view.numel()
        self.half_targets[id(master)] = half_view
        self._flat = None

    # ------------------------------------------------------------------ state
    def _init_state(self, p):
        st = self.state[p]
        if self.state_bits == 8:
            return self._init_state8(p, st)
        if len(st) == 0:
            st["step"] = torch.zeros((), dtype=torch.float32)
            st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
        return st

    def _init_state8(self, p, st):
        if len(st) == 0:
            st["step"] = torch.zeros((), dtype=torch.float32)
        for key in ("exp_avg", "exp_avg_sq"):
            if key not in st:
                st[key] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                st[key + "_exponents"] = torch.zeros((p.numel() + 127) // 128, dtype=torch.uint8, device=p.device)
            elif st[key].dtype != torch.uint8:  # loaded from a checkpoint
                from nanotron_b200 import ops

                st[key], st[key + "_exponents"] = ops.q8_encode(st[key].to(p.device, torch.float32).contiguous().view(p.shape), signed=key == "exp_avg")
        return st

    def state_dict(self):
        """As ``torch.optim.AdamW`` gives it; 8-bit states appear as the fp32 values they stand for."""
        sd = super().state_dict()
        if self.state_bits == 8:
            from nanotron_b200 import ops

            def decoded(st):
                out = {k: v for k, v in st.items() if not k.endswith("_exponents")}
                for key in ("exp_avg", "exp_avg_sq"):
                    if key + "_exponents" in st and st[key].dtype == torch.uint8:
                        out[key] = ops.q8_decode(st[key], st[key + "_exponents"], signed=key == "exp_avg")
                return out

            sd["state"] = {k: decoded(st) if isinstance(st, dict) else st for k, st in sd["state"].items()}
        return sd

    def _try_build_flat_plan(self):
        """All params must tile one contiguous fp32 range in address order, with constant grad / half offsets."""
        items = []
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                items.append((p, gi))
        if not items or not items[0][0].is_cuda or any(p.dtype != torch.float32 or not p.is_contiguous() for p, _ in items):
            return None
        items.sort(key=lambda it: it[0].data_ptr())
        first = items[0][0]
        base = first.data_ptr()
        gbase = first.grad.data_ptr()
        h0 = self.half_targets.get(id(first))
        use_half = h0 is not None
        hbase = h0.data_ptr() if use_half else 0
        storage_end = first.untyped_storage().data_ptr() + first.untyped_storage().nbytes()
        segs = []
        cursor = 0  # elements from base
        for p, gi in items:
            off = (p.data_ptr() - base) // 4
            if (p.data_ptr() - base) % 4 or off < cursor or off - cursor >= 128:
                return None  # gaps larger than the alignment padding: not one flat range
            g = p.grad
            if g.dtype != torch.float32 or not g.is_contiguous() or g.data_ptr() - gbase != p.data_ptr() - base:
                return None
            h = self.half_targets.get(id(p))
            if use_half != (h is not None):
                return None
            if use_half and (h.dtype != torch.bfloat16 or (h.data_ptr() - hbase) * 2 != p.data_ptr() - base):
                return None
            cursor = off + p.numel()
            segs.append((cursor, gi))
        total = (cursor + 3) // 4 * 4
        if base + total * 4 > storage_end or base % 16 or gbase % 16 or (use_half and hbase % 8):
            return None
        # merge neighbouring segments of the same group; padding elements between parameters take the hyper-parameters
        # of the following segment (they are zeros and stay zeros: zero grad, zero weight)
        merged = []
        for end, gi in segs:
            if merged and merged[-1][1] == gi:
                merged[-1] = (end, gi)
            else:
                merged.append((end, gi))
        merged[-1] = (total, merged[-1][1])
        dev = first.device
        flat_p = torch.as_strided(first, (total,), (1,), storage_offset=first.storage_offset())
        flat_g = torch.as_strided(first.grad, (total,), (1,), storage_offset=first.grad.storage_offset())
        flat_h = torch.as_strided(h0, (total,), (1,), storage_offset=h0.storage_offset()) if use_half else None
        # states: adopt existing values, then re-home them in flat buffers
        flat_m = torch.zeros(total, dtype=torch.float32, device=dev)
        flat_v = torch.zeros(total, dtype=torch.float32, device=dev)
        for p, _ in items:
            st = self._init_state(p)
            off = (p.data_ptr() - base) // 4
            for key, flat in (("exp_avg", flat_m), ("exp_avg_sq", flat_v)):
                view = flat[off : off + p.numel()].view(p.shape)
                view.copy_(st[key].to(dev))
                st[key] = view
        return {
            "p": flat_p, "g": flat_g, "h": flat_h, "m": flat_m, "v": flat_v, "items": items,
            "seg_end": torch.tensor([e for e, _ in merged], dtype=torch.int64, device=dev),
            "seg_group": [gi for _, gi in merged],
            "seg_lr": torch.empty(len(merged), dtype=torch.float32, device=dev),
            "seg_wd": torch.tensor([float(self.param_groups[gi]["weight_decay"]) for _, gi in merged], dtype=torch.float32, device=dev),
            "lr_cache": None,
        }

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        from nanotron_b200 import ops

        first = next((p for g in self.param_groups for p in g["params"]), None)
        if self.state_bits == 8:
            self._step8()
            return loss
        if first is not None and first.is_cuda and ops.get_mode() != "torch" and not self._flat_failed:
            if self._flat is None:
                self._flat = self._try_build_flat_plan()
                self._flat_failed = self._flat is None
            if self._flat is not None:
                self._flat_step()
                return loss
        self._per_tensor_step()
        return loss

    def _flat_step(self):
        from nanotron_b200.ops import native

        plan = self._flat
        lrs = tuple(float(self.param_groups[gi]["lr"]) for gi in plan["seg_group"])
        if plan["lr_cache"] != lrs:
            plan["seg_lr"].copy_(torch.tensor(lrs, dtype=torch.float32), non_blocking=True)
            plan["lr_cache"] = lrs
        step_val = None
        for p, _ in plan["items"]:
            st = self.state[p]
            st["step"] += 1
            step_val = float(st["step"])
        g0 = self.param_groups[plan["seg_group"][0]]
        beta1, beta2 = g0["betas"]
        native.adamw_flat(plan["p"], plan["g"], plan["m"], plan["v"], plan["h"], plan["seg_end"], plan["seg_lr"], plan["seg_wd"], beta1, beta2, g0["eps"], step_val, self.grad_scale)
        if plan["h"] is not None:
            for p, _ in plan["items"]:
                p._half_written = True

    def _step8(self):
        """All tensors of a device with the same hyper-parameters and step number in one call (on CUDA one launch)."""
        from nanotron_b200 import ops

        calls = {}
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self._init_state(p)
                st["step"] += 1
                calls.setdefault((tuple(group["betas"]), group["eps"], float(st["step"]), p.device), []).append((p, st, float(group["lr"]), float(group["weight_decay"])))
        for (betas, eps, step, device), items in calls.items():
            ps = [p for p, *_ in items]
            targets = [self.half_targets.get(id(p)) for p in ps]
            halves = [h if h is not None and h.dtype == torch.bfloat16 and h.is_contiguous() else None for h in targets]
            ops.adamw_multi_tensor(
                ps, [p.grad for p in ps], [st["exp_avg"] for _, st, *_ in items], [st["exp_avg_sq"] for _, st, *_ in items],
                exp_avg_exponents=[st["exp_avg_exponents"] for _, st, *_ in items], exp_avg_sq_exponents=[st["exp_avg_sq_exponents"] for _, st, *_ in items],
                halves=halves, lr=[lr for *_, lr, _ in items], weight_decay=[wd for *_, wd in items], beta1=betas[0], beta2=betas[1], eps=eps, step=step,
                grad_scale=self._scale_on(device), seed=ref.mix32((self.state_seed * 0x9E3779B9 + int(step)) & 0xFFFFFFFF),
            )
            for p, target, written in zip(ps, targets, halves):
                if target is None:
                    continue
                if written is None:  # fp16 or fp32 copies
                    target.copy_(p.view(-1))
                p._half_written = True

    def _scale_on(self, device):
        return None if self.grad_scale is None else torch.as_tensor(self.grad_scale, dtype=torch.float32, device=device)

    def _per_tensor_step(self):
        from nanotron_b200 import ops

        for group in self.param_groups:
            beta1, beta2 = group["betas"]
            lr = float(group["lr"])
            together, alone = {}, []  # (step number, device) -> tensors that the multi-tensor kernel takes; the others
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self._init_state(p)
                st["step"] += 1
                item = (p, p.grad, st["exp_avg"], st["exp_avg_sq"], self.half_targets.get(id(p)))
                if p.is_cuda and ops.get_mode() != "torch" and self._multi_tensor_takes(*item):
                    together.setdefault((float(st["step"]), p.device), []).append(item)
                else:
                    alone.append((float(st["step"]), item))
            for (step_val, device), items in together.items():
                ps, gs, ms, vs, halves = (list(x) for x in zip(*items))
                ops.adamw_multi_tensor(ps, gs, ms, vs, lr=lr, beta1=beta1, beta2=beta2, eps=group["eps"], weight_decay=group["weight_decay"], step=step_val, halves=halves, grad_scale=self._scale_on(device))
            scale = float(self.grad_scale) if alone and self.grad_scale is not None else 1.0
            for step_val, (p, g, m, v, h) in alone:
                if p.dtype == torch.float32:
                    ref.adamw_step(p, g.float(), m, v, lr, beta1, beta2, group["eps"], group["weight_decay"], step_val, grad_scale=scale)
                else:
                    pf, mf, vf = p.float(), m.float(), v.float()
                    ref.adamw_step(pf, g.float(), mf, vf, lr, beta1, beta2, group["eps"], group["weight_decay"], step_val, grad_scale=scale)
                    p.copy_(pf), m.copy_(mf), v.copy_(vf)
                if h is not None:
                    h.copy_(p.view(-1))
            for p, _, _, _, h in [it for items in together.values() for it in items] + [it for _, it in alone]:
                if h is not None:
                    p._half_written = True

    @staticmethod
    def _multi_tensor_takes(p, g, m, v, h) -> bool:
        return (
            p.dtype == torch.float32 and g.dtype in (torch.float32, torch.bfloat16) and m.dtype == v.dtype == torch.float32
            and p.is_contiguous() and m.is_contiguous() and v.is_contiguous() and g.device == m.device == v.device == p.device
            and (h is None or (h.dtype == torch.bfloat16 and h.is_contiguous()))
        )
