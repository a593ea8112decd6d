"""Learning on the GPU from self-play samples: what the reference's training step does (train.jl:47-125; losses :12-15, optimiser :50) for the
snetwork2 that the engine plays with, with the operators of alphagpu_amd.ops: every layer a product in 8 bits, forward and backward, the
policy loss on log_probs, one AdamW step over all weights.

    learner = Learner(net)                        # net: SNetwork2
    learner.train(buffer, steps=100, batch=4096)  # buffer: PoolSample
    engine.set_network(learner.network())

The reference's third head (features of the final position, weight 0.001) is dropped by convert_back (DenseNet.jl:331-333) and is not learnt here, and its
weight decay is added to the gradient where AdamW's is not.
"""
import numpy as np
import torch

from . import ops
from .net import SNetwork2


class Learner:
    """The network's weights in float32 on a GPU, and the state of their optimiser.

    net: SNetwork2 to start from.  bits: 32 or 8, the optimiser's states.  lr, betas, eps, weight_decay, seed, capturable: as in ops.AdamW."""

    def __init__(self, net, device=0, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-4, bits=32, seed=0, capturable=False):
        self.H, self.T, self.A, self.inp = net.H, net.T, net.A, net.inp
        self.device = torch.device("cuda", device)

        def matrix(flat, rows, cols):                        # Flux memory order W[o + out i] -> [out, in]
            return torch.from_numpy(np.asarray(flat, np.float32).reshape(cols, rows).T.copy()).to(self.device)

        H, T, A = self.H, self.T, self.A
        self.W0 = matrix(net.W0, H, self.inp)
        self.Wres = [matrix(net.Wres[t * H * H:(t + 1) * H * H], H, H) for t in range(T)]
        self.Whead = torch.cat([matrix(net.Wp, A, H), matrix(net.Wv, 1, H)])                 # policy and value heads are one product
        self.bhead = torch.from_numpy(np.concatenate([net.bp, net.bv]).astype(np.float32)).to(self.device)
        self.params = [self.W0, *self.Wres, self.Whead, self.bhead]
        for p in self.params:
            p.requires_grad_()
        self.optimiser = ops.AdamW(self.params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, seed=seed, capturable=capturable)

    def forward(self, planes, params=None):
        """planes [n, 2 VS] (any number type) -> (policy logits [n, A], value before the sigmoid [n]), float32; DenseNet.jl:294-304.
        params: other tensors in the place of self.params."""
        if planes.dim() != 2 or planes.shape[1] != self.inp or planes.device != self.device:
            raise ValueError(f"planes: [n, {self.inp}] on {self.device}, not {list(planes.shape)} on {planes.device}")
        first, *res, head, bias = self.params if params is None else params
        h = ops.linear_fp8(planes.to(torch.bfloat16), first, relu=True)
        for w in res:
            h = h + ops.linear_fp8(h, w, relu=True)          # (both terms are >= 0: the relu around the sum changes nothing)
        y = ops.linear_fp8(h.float(), head, bias)
        return y[:, :self.A], y[:, self.A]

    def gradients(self, planes, policy, value, mask=None):
        """The losses of every sample (policy [n]: cross entropy against the search's policy [n, A]; value [n]: squared error of the sigmoid against
        value [n]) and the gradients of their mean sum."""
        # leaves of their own: a graph that somebody else has recorded over the weights (on another stream, perhaps) has no part in this backward pass, which
        # may be under capture
        leaves = [p.detach().requires_grad_() for p in self.params]
        logits, v = self.forward(planes, leaves)
        r = ops.log_probs(logits, mask=mask, target=policy)
        with torch.no_grad():                                # the mean's cotangents, written out: nothing here adds up over the batch
            n = max(planes.shape[0], 1)
            s = torch.sigmoid(v)
            off = s - value
            g_value = off * s * (1 - s) * (2 / n)
            g_policy = torch.full_like(r.target, -1 / n)
        grads = torch.autograd.grad([r.target, v], leaves, [g_policy, g_value])
        return -r.target.detach(), off * off, list(grads)

    def step(self, planes, policy, value, mask=None):
        """One step on a batch of samples in device memory -> (policy loss [n], value loss [n]) of the weights before it."""
        policy_loss, value_loss, grads = self.gradients(planes, policy, value, mask)
        self.optimiser.step(grads)
        return policy_loss, value_loss

    def train(self, buffer, steps, batch, seed=0):
        """`steps` steps on random batches of a PoolSample (train.jl:47-125) -> mean (policy loss, value loss) of each step, [steps, 2] numpy."""
        n = buffer.length_buffer()
        if n < 1:
            raise ValueError("train: the buffer is empty")
        rng, losses = np.random.default_rng(seed), []
        for _ in range(int(steps)):
            at = rng.integers(0, n, int(batch))
            put = lambda a: torch.from_numpy(np.ascontiguousarray(a[at])).to(self.device)  # noqa: E731
            p, v = self.step(put(buffer.state), put(buffer.policy), put(buffer.value))
            losses.append(torch.stack([p.mean(), v.mean()]))
        return torch.stack(losses).cpu().numpy() if losses else np.zeros((0, 2), np.float32)

    def network(self):
        """The weights as an SNetwork2 (host memory), for Engine.set_network."""
        out = SNetwork2.__new__(SNetwork2)
        out.inp, out.H, out.T, out.A = self.inp, self.H, self.T, self.A
        flat = lambda w: np.ascontiguousarray(w.detach().t().contiguous().cpu().numpy().reshape(-1))  # noqa: E731
        out.W0 = flat(self.W0)
        out.Wres = np.concatenate([flat(w) for w in self.Wres]) if self.T else np.zeros(self.H * self.H, np.float32)
        out.Wp, out.Wv = flat(self.Whead[:self.A]), flat(self.Whead[self.A:])
        b = self.bhead.detach().cpu().numpy()
        out.bp, out.bv = b[:self.A].copy(), b[self.A:].copy()
        return out


__all__ = ["Learner"]
