"""Inputs and 64-bit references for the packed attention sublayer's operators
(beatlm_amd.ops): plain torch on the tensors' device, from the formulas of
include/beatlm_ops.h, with the magnitudes that the tolerances are made of.

Tolerances. A value rounded once to type t is off by at most half a step,
u(t) = finfo(t).eps / 2 relative. The operators keep f32 inside, so beside the
output's rounding an element carries the f32 errors of its sums (each product
and addition 2^-24 of the magnitudes summed), and attention on 16-bit types
the rounding of the probabilities and of the scores' gradients to the type
for the matrix products: u(t) of the sum's magnitude.
"""

import math

import torch

from beatlm_amd import hip, ops

F32 = 2.0**-24

DTYPES = {"f32": (torch.float32, hip.F32), "f16": (torch.float16, hip.F16), "bf16": (torch.bfloat16, ops.BF16)}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, tol, what):
    """Element by element; infinities have to be the same."""
    got, want = got.double(), want.double()
    same = got == want  # infinities among them
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    bad = ~(off <= tol)
    if bool(bad.any()):
        at = int(bad.flatten().nonzero()[0])
        worst = (off / tol.clamp(min=1e-300)).flatten()
        raise AssertionError(
            f"{what}: {int(bad.sum())} of {bad.numel()} beyond the tolerance, first at {at}: got {float(got.flatten()[at])}, "
            f"want {float(want.flatten()[at])} +- {float(tol.expand_as(off).flatten()[at])}; worst {float(worst.max()):.3g} times it")


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------


class Packed:
    """One packed attention problem on the GPU: documents of (queries, keys),
    tensors with spare rows, their rows and heads strided by `layout`
    ("plain", "qkv": three views of one tensor, "heads": [heads][rows][d]),
    garbage (NaN) everywhere that no document owns."""

    def __init__(self, lens, dtype, q_heads, kv_heads, d, mask="none", cap=0.0, bias=None, axes=0, layout="plain", gap=0, seed=1,
                 scale=None, prefix=None, spread=1.0):
        self.torch_dtype, self.dtype = DTYPES[dtype]
        self.lens, self.q_heads, self.kv_heads, self.d = lens, q_heads, kv_heads, d
        self.mask, self.cap, self.axes, self.gap = mask, cap, axes, gap
        self.scale = d**-0.5 if scale is None else scale
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.q_offsets, self.k_offsets = [gap], [gap]  # rows before the first document too
        for n_q, n_k in lens:
            self.q_offsets.append(self.q_offsets[-1] + n_q)
            self.k_offsets.append(self.k_offsets[-1] + n_k)
        self.q_rows, self.k_rows = self.q_offsets[-1] + gap, self.k_offsets[-1] + gap

        def tensor(rows, heads, fill):
            if layout == "heads":
                t = torch.full((heads, rows, d), fill, device="cuda", dtype=self.torch_dtype).permute(1, 0, 2)
            elif layout == "qkv":
                t = torch.full((rows, heads + 3, d + 8), fill, device="cuda", dtype=self.torch_dtype)[:, 1:1 + heads, :d]
            else:
                t = torch.full((rows, heads, d), fill, device="cuda", dtype=self.torch_dtype)
            return t

        def random(rows, heads, size):
            t = tensor(rows, heads, math.nan)
            t[gap:rows - gap] = (torch.randn(rows - 2 * gap, heads, d, generator=g, device="cuda") * size).to(self.torch_dtype)
            return t

        self.q, self.d_out = random(self.q_rows, q_heads, spread), random(self.q_rows, q_heads, 1.0)
        self.k, self.v = random(self.k_rows, kv_heads, 1.0), random(self.k_rows, kv_heads, 1.0)
        self.SENTINEL = 7.0
        self.out, self.d_q = (tensor(self.q_rows, q_heads, self.SENTINEL) for _ in range(2))
        self.d_k, self.d_v = (tensor(self.k_rows, kv_heads, self.SENTINEL) for _ in range(2))
        self.lse = torch.full((q_heads, self.q_rows), self.SENTINEL, device="cuda")
        ints = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
        self.q_off, self.k_off = ints(self.q_offsets), ints(self.k_offsets)
        self.prefixes = prefix if prefix is not None else [n_k // 3 for _, n_k in lens]
        self.prefix = ints(self.prefixes) if mask == "prefix" else None
        self.slopes = self.d_slopes = self.q_positions = self.k_positions = None
        if bias:
            self.slopes = (torch.rand(q_heads, generator=g, device="cuda") * bias).contiguous()
            self.d_slopes = torch.full((q_heads,), self.SENTINEL, device="cuda")
        if axes:
            place = lambda n: torch.randint(-40, 40, (n, axes), generator=g, device="cuda", dtype=torch.int32)  # noqa: E731
            self.q_positions, self.k_positions = place(self.q_rows), place(self.k_rows)

    def args(self, ctx, backward, max_keys=0):
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        heads = lambda t: ops.Heads(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
        a = ops.AttentionArgs(
            dtype=self.dtype, q_heads=self.q_heads, kv_heads=self.kv_heads, head_dim=self.d, q_rows=self.q_rows, k_rows=self.k_rows,
            documents=len(self.lens), mask={"none": 0, "causal": 1, "prefix": 2}[self.mask], axes=self.axes, max_keys=max_keys,
            scale=self.scale, softcap=self.cap, q_offsets=at(self.q_off), k_begin=at(self.k_off), k_end=self.k_off.data_ptr() + 4,
            prefix=at(self.prefix), slopes=at(self.slopes), q_positions=at(self.q_positions), k_positions=at(self.k_positions),
            q=heads(self.q), k=heads(self.k), v=heads(self.v), out=heads(self.out), lse=at(self.lse))
        n = ops.attention_workspace(ctx, a, backward)
        # what the workspace holds before a call means nothing
        self.workspace = torch.full((n + 16,), 0xFF, device="cuda", dtype=torch.uint8)
        a.workspace, a.workspace_bytes = self.workspace.data_ptr(), n
        return a

    def grads(self):
        heads = lambda t: ops.Heads(t.data_ptr(), t.stride(0), t.stride(1))  # noqa: E731
        return ops.AttentionGrads(d_out=heads(self.d_out), d_q=heads(self.d_q), d_k=heads(self.d_k), d_v=heads(self.d_v),
                                  d_slopes=None if self.d_slopes is None else self.d_slopes.data_ptr())

    def reference(self, backward):
        """{name: (value, tolerance)} in 64 bits, the untouched rows among them."""
        u = half_step(self.torch_dtype)
        inner = 0.0 if self.torch_dtype == torch.float32 else u  # P and dS rounded for the products
        got = {}

        def put(name, like):
            got[name] = (torch.full(like.shape, self.SENTINEL, device="cuda", dtype=torch.float64),
                         torch.zeros(like.shape, device="cuda", dtype=torch.float64))
            return got[name]

        out, lse = put("out", self.out), put("lse", self.lse)
        if backward:
            d_q, d_k, d_v = put("d_q", self.d_q), put("d_k", self.d_k), put("d_v", self.d_v)
            for t in (d_k, d_v):
                t[0][self.k_offsets[0]:self.k_offsets[-1]] = 0.0
            if self.slopes is not None:
                d_slopes = put("d_slopes", self.d_slopes)
                d_slopes[0].zero_()
        group = self.q_heads // self.kv_heads
        for doc, (n_q, n_k) in enumerate(self.lens):
            rows = slice(self.q_offsets[doc], self.q_offsets[doc + 1])
            keys = slice(self.k_offsets[doc], self.k_offsets[doc + 1])
            at = torch.arange(n_q, device="cuda")[:, None] + (n_k - n_q)
            j = torch.arange(n_k, device="cuda")[None]
            seen = torch.ones(n_q, n_k, device="cuda", dtype=torch.bool)
            if self.mask != "none":
                seen = j <= at
            if self.mask == "prefix":
                seen = seen | (j < self.prefixes[doc])
            far = (at - j).abs().double()
            if self.axes:
                far = (self.q_positions[rows].double()[:, None] - self.k_positions[keys].double()[None]).abs().sum(-1)
            for h in range(self.q_heads):
                kv = h // group
                q, k, v = self.q[rows, h].double(), self.k[keys, kv].double(), self.v[keys, kv].double()
                raw = q @ k.T * self.scale
                size = q.abs() @ k.abs().T * abs(self.scale)
                s = self.cap * torch.tanh(raw / self.cap) if self.cap else raw
                slope = float(self.slopes[h]) if self.slopes is not None else 0.0
                s = (s - slope * far).masked_fill(~seen, -math.inf)
                # what one score may be off: the product's sum, the cap (a tanh good to a few
                # steps of 1, times the cap), the bias, and the exponent's argument in base two
                off = F32 * ((self.d + 4) * size + 8 * self.cap + 4 * slope * far + 4 * s.masked_fill(~seen, 0.0).abs() + 8)
                off = off.masked_fill(~seen, 0.0)
                worst = off.amax(1) if n_k else torch.zeros(n_q, device="cuda", dtype=torch.float64)
                stat = torch.logsumexp(s, 1) if n_k else torch.full((n_q,), -math.inf, device="cuda", dtype=torch.float64)
                dead = stat == -math.inf
                p = torch.where(seen, (s - stat.masked_fill(dead, 0.0)[:, None]).exp(), torch.zeros_like(s))
                relative = 2 * (off + worst[:, None] + F32 * (n_k + 16))  # of each probability
                o = p @ v
                out[0][rows, h] = o
                out[1][rows, h] = u * o.abs() + (p * (relative + inner)) @ v.abs() + 1e-30
                if self.torch_dtype == torch.float16:  # its own subnormals, and those of P
                    out[1][rows, h] += 2.0**-25 * (1 + seen.double() @ v.abs())
                lse[0][h, rows] = stat
                lse[1][h, rows] = worst + F32 * (n_k + 16 + 4 * stat.masked_fill(dead, 0.0).abs())
                if not backward:
                    continue
                g = self.d_out[rows, h].double()
                dp = g @ v.T
                dp_size = g.abs() @ v.abs().T
                delta = (p * dp).sum(1, keepdim=True)
                # delta comes from the rounded output, or from the row's own products
                delta_off = (g.abs() * out[1][rows, h]).sum(1, keepdim=True) + F32 * (self.d + 8) * (p * dp_size).sum(1, keepdim=True)
                t = torch.tanh(raw / self.cap) if self.cap else torch.zeros_like(raw)
                slack = 1 - t * t
                ds = p * (dp - delta)
                ds_off = p * (relative * (dp - delta).abs() + F32 * (self.d + 8) * dp_size + delta_off)
                inner_s = ds * slack * self.scale
                # 1 - tanh^2 is off by a few steps of 1 and by twice the score's error over the cap
                inner_off = abs(self.scale) * (ds_off * slack + ds.abs() * (16 * F32 + (4 * off / self.cap if self.cap else 0.0)))
                inner_off = inner_off + inner * inner_s.abs()
                tiny = 0.0
                if self.torch_dtype == torch.float16:
                    # Operands below f16's smallest normal number, 2^-14, are off by half its
                    # smallest step, 2^-25: P itself, and dS divided by a power of two that is
                    # at most the largest |dO| of the key head's rows.
                    tiny = 2.0**-25
                    heads = self.d_out[:, kv * group:(kv + 1) * group].double().nan_to_num(0.0)
                    inner_off = inner_off + abs(self.scale) * tiny * heads.abs().max() * seen
                d_q[0][rows, h] = inner_s @ k
                d_q[1][rows, h] = u * d_q[0][rows, h].abs() + (inner_off + F32 * (n_k + 8) * inner_s.abs()) @ k.abs() + 1e-30
                d_k[0][keys, kv] += inner_s.T @ q
                d_k[1][keys, kv] += (inner_off + F32 * (group * n_q + 8) * inner_s.abs()).T @ q.abs()
                d_v[0][keys, kv] += p.T @ g
                d_v[1][keys, kv] += (p * (relative + inner + F32 * (group * n_q + 8)) + tiny * seen).T @ g.abs()
                if self.slopes is not None:
                    d_slopes[0][h] -= (ds * far).sum()
                    # through the row's own sums in f32: sum P dP far - (sum P dP)(sum P far)
                    row_far = (p * far).sum(1, keepdim=True)
                    own = relative + F32 * (n_k + self.d + 16)
                    d_slopes[1][h] += ((own * p * dp_size * far).sum() + (own * p * dp_size * row_far).sum()
                                       + (own * p * far * delta.abs()).sum() + F32 * self.q_rows * (ds.abs() * far).sum()) + 1e-30
        if backward:
            half = 2.0**-25 if self.torch_dtype == torch.float16 else 0.0
            inside = slice(self.k_offsets[0], self.k_offsets[-1])
            for t in (d_k, d_v):
                t[1][inside] += u * t[0][inside].abs() + half + 1e-30
            d_q[1][self.q_offsets[0]:self.q_offsets[-1]] += half
        return got

    def check(self, names, backward):
        want = self.reference(backward)
        for name in names:
            value = getattr(self, name)
            if value is not None:
                assert_within(value, *want[name], name)
