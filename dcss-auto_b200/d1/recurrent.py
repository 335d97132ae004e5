"""A joint-action head with a memory, on the conv policy's features, trained by reinforcement.

    head = RecurrentHead(seed=0)
    state = head.state(n)
    joint, logp, state = head.act(h, env.legal, state, reset=ended, generator=g)    # one decision
    loss = head.update(hs, joints, legals, logps, advantages, first, resets)        # a rollout [T, n]

    features h (bf16 [T, n, 512])
      gates and inputs of 256 channels              (tcgen05 GEMM, d1_gemm)
      memory: h_t = a_t h_{t-1} + (1 - a_t) x_t     (d1.gated_scan, cut where an episode begins)
      layer norm                                    (d1.layer_norm)
      28 joint actions: verb and target             (tcgen05 GEMM)
      log p(joint), entropy                         (d1.token_logprob, joint legal bits)
      clipped policy loss, KL and entropy terms     (d1.policy_loss)

The conv policy sees a window of the map around the player; what has left it is only in
the memory. update() goes back through the same operators and ends with d1.muon over the
weight matrices (the gates' and the inputs' are two of a stack) and d1.adamw over the
vectors, at one rate. Masters are fp32, the GEMM operands bf16 copies that Muon refreshes. The
joint actions are d1.imitation's.
"""
import torch

from . import gemm as G
from ._lib import check, launch_stream, library, resolve_device
from .adamw import AdamW
from .conv_policy import WIDTH
from .gated_scan import gated_scan, gated_scan_backward
from .imitation import JOINT, PITCH, joint_legal
from .layer_norm import layer_norm, layer_norm_backward
from .muon import Muon
from .policy_loss import policy_loss
from .token_logprob import token_logprob, token_logprob_backward

F32, BF16 = torch.float32, torch.bfloat16
MEMORY = 256


class RecurrentHead:
    def __init__(self, device='cuda', seed=0, lr=3e-4, weight_decay=0.01, clip=0.2, kl_coef=0.0, ent_coef=0.01, memory=MEMORY):
        if memory < 8 or memory % 8:
            raise ValueError('memory must be a multiple of 8 channels')
        self.device = dev = resolve_device(device)
        g = torch.Generator(device='cpu').manual_seed(seed)
        normal = lambda *s: torch.randn(*s, generator=g, dtype=F32) / s[-1] ** 0.5
        out = torch.zeros(PITCH, memory, dtype=F32)
        out[:JOINT] = normal(JOINT, memory)
        bias = torch.zeros(2 * memory, dtype=F32)
        bias[:memory] = torch.linspace(0.0, 5.0, memory, dtype=F32)  # time constants from 2 to 150 decisions
        self.memory = memory
        self.params = {'in': normal(2, memory, WIDTH), 'out': out, 'in_b': bias, 'out_b': torch.zeros(PITCH, dtype=F32),
                       'norm_w': torch.ones(memory, dtype=F32), 'norm_b': torch.zeros(memory, dtype=F32)}
        self.params = {k: p.to(dev) for k, p in self.params.items()}
        self.grads = {k: torch.zeros_like(p) for k, p in self.params.items()}
        self.w = {k: self.params[k].to(BF16) for k in ('in', 'out')}
        self.clip, self.kl_coef, self.ent_coef = clip, kl_coef, ent_coef
        pick = lambda d, names: [d[k] for k in names]
        matrices, vectors = ('in', 'out'), ('in_b', 'out_b', 'norm_w', 'norm_b')
        self.muon = Muon(pick(self.params, matrices), pick(self.grads, matrices), lr=lr, weight_decay=weight_decay,
                         copies=pick(self.w, matrices))
        self.adamw = AdamW(pick(self.params, vectors), pick(self.grads, vectors), lr=lr, weight_decay=0.0)
        self.lib = library()

    def state(self, n):
        """The memory of n environments that have seen nothing (float32 [n, memory])."""
        return torch.zeros((n, self.memory), dtype=F32, device=self.device)

    def forward(self, h, state, reset=None):
        """(logits [T * n, 28], the memory after the last step, what the backward pass needs)
        of features h (bf16 [T, n, 512]); reset (bool [T, n]): an episode begins at that step."""
        T, n, _ = h.shape
        p, m = self.params, self.memory
        proj = G.gemm(h.reshape(T * n, WIDTH), self.w['in'].view(2 * m, WIDTH), bias=p['in_b']).view(T, n, 2 * m)
        gate, x = proj[..., :m], proj[..., m:]
        y, last = gated_scan(x, gate, state, reset=reset)
        z, mean, rstd = layer_norm(y, p['norm_w'], p['norm_b'])
        logits = G.gemm(z.view(T * n, m), self.w['out'], bias=p['out_b'])[:, :JOINT]
        return logits, last, (h, x, gate, y, z, mean, rstd, state, reset)

    def act(self, h, legal, state, reset=None, generator=None):
        """One decision: actions drawn among the legal ones (int64 [n]) for features h (bf16 [n, 512]),
        their log-probabilities and the memory after it."""
        logits, last, _ = self.forward(h[None], state, None if reset is None else reset[None])
        bits = joint_legal(legal)
        on = (bits[:, None] >> torch.arange(JOINT, device=self.device, dtype=torch.int32)) & 1 == 1
        noise = torch.empty(logits.shape, dtype=F32, device=self.device).exponential_(generator=generator)
        joint = (logits.float() - noise.log()).masked_fill(~on, -torch.inf).argmax(1)
        return joint, token_logprob(logits, joint, legal=bits).logp, last

    def backward(self, logits, joint, bits, r, loss, saved):
        """Fills self.grads; returns the gradients of the features (bf16 [T, n, 512]) and of the first memory."""
        h, x, gate, y, z, mean, rstd, state, reset = saved
        (T, n, m), g = y.shape, self.grads
        rows = T * n
        dl = torch.zeros((rows, PITCH), dtype=BF16, device=self.device)
        token_logprob_backward(logits, joint, r.stats, r.entropy, loss.dlogp.view(-1), loss.dentropy.view(-1), legal=bits, out=dl[:, :JOINT])
        self._weight_gradient(dl, z.view(rows, m), g['out'])
        torch.sum(dl, 0, dtype=F32, out=g['out_b'])
        dy, dw, db = layer_norm_backward(G.gemm_bkn(dl, self.w['out']).view(T, n, m), y, mean, rstd, self.params['norm_w'])
        g['norm_w'].copy_(dw)
        g['norm_b'].copy_(db)
        dx, dgate, dstate = gated_scan_backward(dy, x, gate, y, state, reset=reset)
        dproj = torch.cat((dgate, dx), 2).view(rows, 2 * m)
        self._weight_gradient(dproj, h.reshape(rows, WIDTH), g['in'].view(2 * m, WIDTH))
        torch.sum(dproj, 0, dtype=F32, out=g['in_b'])
        return G.gemm_bkn(dproj, self.w['in'].view(2 * m, WIDTH)).view(T, n, WIDTH), dstate

    def _weight_gradient(self, d, x, out):
        slabs = torch.empty((G.splits_for(d.shape[0], 8), *out.shape), dtype=F32, device=self.device)
        G.gemm_ex(d, x, a_kn=True, b_kn=True, out_f32=slabs, splits=slabs.shape[0])
        check(self.lib.d1_reduce_slabs(slabs.data_ptr(), slabs.shape[0], out.numel(), out.data_ptr(), launch_stream(self.device)),
              'd1_reduce_slabs')

    def update(self, h, joint, legal, old_logp, advantage, state, reset=None, live=None, ref_logp=None):
        """One step on a rollout: features h (bf16 [T, n, 512]), the actions taken (int64 [T, n]) where
        `legal` (the environments' bits, [T, n]) held, their log-probabilities then, their advantages
        ([T, n], or one for each step [T]), the memory before it. live (bool [T, n]): the decisions that count. Returns the
        PolicyLoss before the step."""
        T, n = joint.shape
        logits, _, saved = self.forward(h, state, reset)
        bits, flat = joint_legal(legal.reshape(-1)), joint.reshape(-1)
        r = token_logprob(logits, flat, legal=bits)
        loss = policy_loss(r.logp.view(T, n), old_logp, advantage, ref_logp=ref_logp, entropy=r.entropy.view(T, n), mask=live,
                           clip=self.clip, kl_coef=self.kl_coef, ent_coef=self.ent_coef)
        self.backward(logits, flat, bits, r, loss, saved)
        self.muon.step()
        self.adamw.step()
        return loss
