"""A head with a matrix for every leaf of a model's router, trained and served on the operators of yggdrasil_amd.ops:

    PYTHONPATH=. python examples/routed_head.py model.bin tokens.i32     # or without arguments: a small synthetic model

The frozen model gives each token's state and the leaf that its last layer took. A shared head in int8 (int8_linear) and the
leaf's own matrix (grouped_matmul) make the logits; token_logprobs gives the loss of the next tokens, its gradient goes back
through the logits into the leaves' matrices. Served, the same head gives the alternatives of the last token."""
import sys
import tempfile

import numpy as np
import torch

from yggdrasil_amd import Yggdrasil, ops, synth


def states_of(model, tokens):
    """tokens (B, T) -> the last layer's states (B T, n) bf16, in [-1, 1], and the leaves (B T) it took."""
    r = model.run(tokens, leaves=True, states=True)
    h = (r["states"][:, :, -1].float() / 127).to(torch.bfloat16)
    return h.reshape(-1, h.shape[-1]), r["leaves"][:, :, -1].reshape(-1)


class RoutedHead:
    def __init__(self, classes, leaves, n, device, seed=0):
        g = torch.Generator("cpu").manual_seed(seed)
        self.q, self.scale = ops.quantize_weight(torch.randn(classes, n, generator=g).to(device) / n ** 0.5)
        self.w = torch.zeros(leaves, classes, n, dtype=torch.bfloat16, device=device, requires_grad=True)

    def logits(self, h, leaves):
        """h (rows, n), the leaf of each row -> (rows, classes) f32"""
        offsets, order = ops.group_rows(leaves, len(self.w))
        return ops.int8_linear(h, self.q, self.scale).float() + ops.grouped_matmul(h, self.w, offsets, order).float()

    def step(self, h, leaves, targets, rate):
        """One step of gradient descent on the mean loss of the targets (-1: none); the loss in nats."""
        logp = ops.token_logprobs(self.logits(h, leaves), targets).logp
        loss = -logp.sum() / (targets >= 0).sum()
        grad, = torch.autograd.grad(loss, self.w)
        with torch.no_grad():
            self.w -= rate * grad
        return loss.detach()

    @torch.no_grad()
    def alternatives(self, h, leaves, top):
        """The most likely next classes of each row, their log-probabilities, and each row's entropy."""
        r = ops.token_logprobs(self.logits(h, leaves), top=top)
        return r.top_ids, r.top_logp, r.entropy


def next_tokens(tokens, device):
    """Each place's next token, -1 at a row's end."""
    t = torch.as_tensor(np.asarray(tokens), dtype=torch.int32, device=device)
    return torch.cat([t[:, 1:], torch.full_like(t[:, :1], -1)], 1).reshape(-1)


def main(path=None, tokens=None, steps=30, rate=2.0):
    with tempfile.TemporaryDirectory() as tmp:
        if path is None:
            spec = synth.KERNEL_CASES[0]
            path = f"{tmp}/m.bin"
            synth.write_model(spec, synth.KERNEL_SEED, path)
            tokens = synth.kernel_tokens(spec.vocab)
        model = Yggdrasil.load(path)
        h, leaves = states_of(model, tokens)
        head = RoutedHead(model.vocab, int(leaves.max()) + 1, h.shape[1], h.device)
        targets = next_tokens(tokens, h.device)
        losses = [head.step(h, leaves, targets, rate) for _ in range(steps)]
        losses = torch.stack(losses).tolist()
        print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} nats a token in {steps} steps")
        last = torch.arange(len(tokens), device=h.device) * np.shape(tokens)[1] + np.shape(tokens)[1] - 1
        ids, logp, entropy = head.alternatives(h[last], leaves[last], 5)
        for i in range(min(len(ids), 4)):
            print(f"stream {i}: entropy {entropy[i]:.2f};", ", ".join(f"{t} {p:.2f}" for t, p in zip(ids[i].tolist(), logp[i].tolist())))
        model.close()
    return losses, ids


if __name__ == "__main__":
    if len(sys.argv) == 3:
        x = np.fromfile(sys.argv[2], np.int32)
        T = min(len(x), 1024)
        main(sys.argv[1], x[:len(x) // T * T].reshape(-1, T))
    else:
        main()
