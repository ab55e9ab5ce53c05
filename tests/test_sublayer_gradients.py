"""How attention's gradients are held against differences of its forward: one
query head's outputs at a time, along directions in which the derivative is the
sum of the |gradient|, so that a wrong sign, factor, head or cap cannot hide in
the tolerance. Shown
here, without a GPU, on the 64-bit forward and on mistakes planted in its
gradients; tests/test_gpu_sublayer_gradients.py holds the kernels' to it."""

import math

import pytest
import torch

# What rounding may add to a difference, of the sum of |gradient| along it: the
# tests of the kernels derive theirs and show that it is less. (A slope is one
# number, whose derivative is small beside the outputs' errors.)
ROUNDING = {"q": 0.05, "k": 0.05, "v": 0.05, "slopes": 0.4}
# Elements move by 2^-6: 32 channels of size 0.8 move a score by some 2^-4.
STEP = 2.0**-6


def plain_forward(q, k, v, lens, scale, mask="none", cap=0.0, slopes=None, prefixes=None):
    """out [rows][heads][d] of packed documents, one head and document at a time."""
    group = q.shape[1] // k.shape[1]
    outs, q0, k0 = [], 0, 0
    for doc, (n_q, n_k) in enumerate(lens):
        at = torch.arange(n_q, device=q.device)[:, None] + (n_k - n_q)
        j = torch.arange(n_k, device=q.device)[None]
        seen = torch.ones(n_q, n_k, device=q.device, dtype=torch.bool) if mask == "none" else j <= at
        if mask == "prefix":
            seen = seen | (j < prefixes[doc])
        heads = []
        for h in range(q.shape[1]):
            s = q[q0:q0 + n_q, h] @ k[k0:k0 + n_k, h // group].T * scale
            s = cap * torch.tanh(s / cap) if cap else s
            s = s if slopes is None else s - slopes[h] * (at - j).abs()
            heads.append(s.masked_fill(~seen, -math.inf).softmax(1) @ v[k0:k0 + n_k, h // group])
        outs.append(torch.stack(heads, 1))
        q0, k0 = q0 + n_q, k0 + n_k
    return torch.cat(outs)


def direction(claimed, head):
    """The signs of what a gradient claims for a head ([rows][heads][channels], or
    one number a head); alternating ones where it claims nothing."""
    part = torch.zeros_like(claimed)
    at = (slice(None), head) if claimed.dim() > 1 else (slice(head, head + 1),)
    part[at] = claimed[at]
    if not bool(part.any()):
        part[at] = (torch.arange(part[at].numel(), device=claimed.device).reshape(part[at].shape) % 2 * 2 - 1).to(claimed)
    return part.sign()


def difference(value, leaf, way, step):
    """(value(leaf + step way) - value(leaf - step way)) / (2 step), from rounded leaves as they are."""
    kept = leaf.clone()
    got = []
    for sign in (1, -1):
        leaf.copy_(kept + sign * step * way)
        got.append(value())
    leaf.copy_(kept)
    return (got[0] - got[1]) / (2 * step)


def truncation(exact, leaf, way):
    """A central difference is off by c h^2, and D(h) - D(h / 2) is 3/4 of that; twice, for what follows it."""
    return 2 * 4 / 3 * abs(difference(exact, leaf, way, STEP) - difference(exact, leaf, way, STEP / 2))


def heads_of(name, head):
    """Where the gradient of a value of one query head's outputs lies: 4 query heads on 2 key heads."""
    return head // 2 if name in ("k", "v") else head


def rejected(name, exact, leaf, claimed, head):
    way = direction(claimed, head)
    slope, along = difference(exact, leaf, way, STEP), float((claimed * way).sum())
    return abs(along - slope) > truncation(exact, leaf, way) + ROUNDING[name] * max(abs(along), abs(slope))


LENS, SCALE, CAP = [(40, 40), (21, 21)], 32**-0.5, 1.5  # scores of size 1 under a cap of 1.5


def problem(device="cpu"):
    g = torch.Generator().manual_seed(5)
    make = lambda *s: torch.randn(*s, generator=g).to(device, torch.float64)  # noqa: E731
    return dict(q=make(61, 4, 32), k=make(61, 2, 32), v=make(61, 2, 32), slopes=torch.tensor([0.02, 0.05, 0.1, 0.2], device=device, dtype=torch.float64)), make(61, 4, 32)


def forward(leaves):
    return plain_forward(leaves["q"], leaves["k"], leaves["v"], LENS, SCALE, "causal", CAP, leaves["slopes"])


def value_of(leaves, d_out, head):
    return lambda: float((forward(leaves)[:, head] * d_out[:, head]).sum())


def gradients(leaves, d_out, head):
    held = {n: t.clone().requires_grad_() for n, t in leaves.items()}
    return dict(zip(held, torch.autograd.grad((forward(held)[:, head] * d_out[:, head]).sum(), list(held.values()))))


NAMES = pytest.mark.parametrize("name", ["q", "k", "v", "slopes"])
HEADS = pytest.mark.parametrize("head", range(4))


@NAMES
@HEADS
def test_right_gradients_pass(name, head):
    leaves, d_out = problem()
    grad = gradients(leaves, d_out, head)[name]
    assert not rejected(name, value_of(leaves, d_out, head), leaves[name], grad, heads_of(name, head))


@NAMES
@HEADS
@pytest.mark.parametrize("factor", [-1.0, 0.5, 2.0, 0.0])
def test_a_wrong_sign_or_factor_or_a_head_left_out_is_rejected(name, head, factor):
    leaves, d_out = problem()
    grad = gradients(leaves, d_out, head)[name] * factor
    assert rejected(name, value_of(leaves, d_out, head), leaves[name], grad, heads_of(name, head))


class Flat(torch.autograd.Function):
    """tanh with a derivative of 1."""

    @staticmethod
    def forward(ctx, x):
        return TANH(x)

    @staticmethod
    def backward(ctx, g):
        return g


TANH = torch.tanh


@pytest.mark.parametrize("name", ["q", "k"])
@HEADS
def test_gradients_without_the_cap_s_derivative_are_rejected(name, head, monkeypatch):
    leaves, d_out = problem()
    monkeypatch.setattr(torch, "tanh", Flat.apply)
    grad = gradients(leaves, d_out, head)[name]
    monkeypatch.undo()
    assert rejected(name, value_of(leaves, d_out, head), leaves[name], grad, heads_of(name, head))
