"""A token mixer of gated delta heads, trained and then served.

One layer: projections, the gated delta rule, a gated group norm over the heads,
an output projection.  The task is recall with overwriting: a step writes a
(key, value) pair, keys come again with other values, and a query step has to
answer with the value that its key was given last; a sum of outer products
cannot forget the earlier ones, the delta rule replaces them.

    python examples/delta_mixer.py [--steps N] [--dtype bfloat16|float32]

trains the layer (gated_delta_forward, group_norm_act_forward and their
backward entry points), then answers the same sequences as a server would: the
prompt in one call that returns the state, the state saved and loaded again,
the rest one token at a time with gated_delta_step, and compares the answers.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir,
                                "triton-ssm_amd"))

import tssm  # noqa: E402
from tssm import session  # noqa: E402


class GatedDelta(torch.autograd.Function):
    """o of gated_delta_forward from a zero state."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta):
        ctx.save_for_backward(q, k, v, g, beta)
        return tssm.gated_delta_forward(q, k, v, g, beta)

    @staticmethod
    def backward(ctx, do):
        return tssm.gated_delta_backward(*ctx.saved_tensors, do.contiguous())[:5]


class GatedNorm(torch.autograd.Function):
    """y of group_norm_act_forward with a weight and a gate."""

    @staticmethod
    def forward(ctx, x, weight, gate, groups):
        y, mean, rstd = tssm.group_norm_act_forward(x, groups, weight, None, gate,
                                                    return_stats=True)
        ctx.save_for_backward(x, weight, gate, mean, rstd)
        ctx.groups = groups
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, gate, mean, rstd = ctx.saved_tensors
        dx, dw, _, dgate = tssm.group_norm_act_backward(dy.contiguous(), x, mean, rstd,
                                                        ctx.groups, weight, None, gate)
        return dx, dw, dgate, None


class DeltaMixer(torch.nn.Module):
    """x [B, L, D] -> [B, L, D]: ``heads`` value heads of K x V states over
    ``key_heads`` key heads.  Parameters and projections are fp32; the delta rule
    and the norm take ``dtype``."""

    def __init__(self, D, key_heads, heads, K, V, dtype):
        super().__init__()
        self.Hk, self.Hv, self.K, self.V, self.dtype = key_heads, heads, K, V, dtype
        self.parts = [key_heads * K, key_heads * K, heads * V, heads * V, heads, heads]
        self.inp = torch.nn.Linear(D, sum(self.parts), bias=False)
        self.out = torch.nn.Linear(heads * V, D, bias=False)
        self.norm = torch.nn.Parameter(torch.ones(heads * V))
        self.decay = torch.nn.Parameter(torch.full((heads,), -4.0))

    def _project(self, x):
        q, k, v, z, a, b = self.inp(x).split(self.parts, dim=-1)
        lead = x.shape[:-1]
        q, k = (F.normalize(t.reshape(*lead, self.Hk, self.K), dim=-1).to(self.dtype)
                for t in (q, k))
        v = F.silu(v).reshape(*lead, self.Hv, self.V).to(self.dtype)
        return q, k, v, -F.softplus(a + self.decay), torch.sigmoid(b), z.to(self.dtype)

    def _finish(self, o, z):
        lead = o.shape[:-2]
        # statistics per token and head: tokens are rows, heads are groups
        y = GatedNorm.apply(o.reshape(-1, self.Hv * self.V), self.norm,
                            z.reshape(-1, self.Hv * self.V).contiguous(), self.Hv)
        return self.out(y.float()).reshape(*lead, -1)

    def forward(self, x):
        q, k, v, g, beta, z = self._project(x)
        return self._finish(GatedDelta.apply(q, k, v, g, beta), z)

    @torch.no_grad()
    def prompt(self, x):
        """x [B, L, D]; also returns the state [B, heads, K, V] that step() goes on from."""
        q, k, v, g, beta, z = self._project(x)
        o, state = tssm.gated_delta_forward(q, k, v, g, beta, return_state=True)
        return self._finish(o, z), state

    @torch.no_grad()
    def step(self, x, state):
        """x [B, D], one token of every stream; the state is updated in place."""
        q, k, v, g, beta, z = self._project(x)
        return self._finish(tssm.gated_delta_step(q, k, v, g, beta, state), z)


class Recall(torch.nn.Module):
    """Embeddings of keys and values, the mixer, and the answers' logits."""

    def __init__(self, keys, values, D=64, key_heads=2, heads=4, K=32, V=32,
                 dtype=torch.bfloat16):
        super().__init__()
        self.key, self.value = torch.nn.Embedding(keys, D), torch.nn.Embedding(values + 1, D)
        self.mixer = DeltaMixer(D, key_heads, heads, K, V, dtype)
        self.answer = torch.nn.Linear(D, values)

    def embed(self, keys, values):
        return self.key(keys) + self.value(values)

    def forward(self, keys, values):
        return self.answer(self.mixer(self.embed(keys, values)))


def recall_batch(B, L, keys, values, generator):
    """(key [B, L], value [B, L], answer [B, L]): a value equal to ``values`` marks
    a query, whose answer is the last value that was written to its key; answers
    elsewhere are -1, and only keys written before are asked for."""
    key = torch.randint(keys, (B, L), generator=generator)
    value = torch.randint(values, (B, L), generator=generator)
    ask = torch.rand(B, L, generator=generator) < 0.4
    held = torch.full((B, keys), -1)
    answer = torch.full((B, L), -1)
    rows = torch.arange(B)
    for t in range(L):
        last = held[rows, key[:, t]]
        ask[:, t] &= last >= 0
        answer[:, t] = torch.where(ask[:, t], last, -1)
        held[rows, key[:, t]] = torch.where(ask[:, t], last, value[:, t])
    return key, value.masked_fill(ask, values), answer


def train(model, steps, B, L, keys, values, generator, lr=3e-3, say=None):
    """Returns the loss of every step."""
    opt = torch.optim.Adam(model.parameters(), lr=lr)
    losses = []
    for i in range(steps):
        key, value, answer = (t.cuda() for t in recall_batch(B, L, keys, values, generator))
        loss = F.cross_entropy(model(key, value).flatten(0, 1), answer.flatten(), ignore_index=-1)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.detach())
        if say and (i + 1) % 50 == 0:
            say(f"step {i + 1}: loss {losses[-1].item():.4f}")
    return torch.stack(losses).tolist()


@torch.no_grad()
def serve(model, key, value, prompt):
    """Logits [B, L, values] with the first ``prompt`` tokens in one call, the
    state through a session's bytes, and every further token by itself."""
    x = model.embed(key, value)
    y, state = model.mixer.prompt(x[:, :prompt])
    saved = session.dumps({"delta": state}, {"tokens": prompt})
    tensors, _ = session.loads(saved, device=x.device)
    state = tensors["delta"]
    ys = [y] + [model.mixer.step(x[:, t], state).unsqueeze(1) for t in range(prompt, x.shape[1])]
    return model.answer(torch.cat(ys, 1))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--dtype", choices=["bfloat16", "float32"], default="bfloat16")
    args = ap.parse_args()
    keys, values, B, L = 24, 32, 64, 96
    torch.manual_seed(0)
    generator = torch.Generator().manual_seed(1)
    model = Recall(keys, values, dtype=getattr(torch, args.dtype)).cuda()
    train(model, args.steps, B, L, keys, values, generator, say=lambda s: print(s, flush=True))
    key, value, answer = (t.cuda() for t in recall_batch(B, L, keys, values, generator))
    with torch.no_grad():
        whole = model(key, value)
    served = serve(model, key, value, L // 2)
    asked = answer >= 0
    for name, logits in (("whole sequences", whole), ("prompt and steps", served)):
        right = (logits.argmax(-1) == answer)[asked].float().mean().item()
        print(f"{name}: {100 * right:.1f}% of {int(asked.sum())} queries right")
    print(f"largest difference of logits: {(whole - served).abs().max().item():.2e} "
          f"of {whole.abs().max().item():.1f}")


if __name__ == "__main__":
    main()
