"""A joint-action head on the conv policy's features, trained on given actions.

    head = JointHead(seed=0)
    pol.encode(env.state, n, buf); pol.features(buf, n)      # ConvPolicy: buf['h']
    out = head.update(buf['h'], joint, env.legal)            # one step towards the actions `joint`

    features h (bf16 [n, 512])
      layer norm                                  (d1.layer_norm)
      28 joint actions: verb and target           (tcgen05 GEMM, d1_gemm)
      log p(joint), entropy, likeliest actions    (d1.token_logprob, joint legal bits)

The loss is -mean(log p(joint)) - ent_coef * mean(entropy) over the rows; the
step goes back through the same operators and ends with d1.adamw over the four
parameter tensors, whose moments are held in 8 bits by default. The joint
actions are the autoregressive head's (9 * verb + target for MOVE and ATTACK,
16 + verb for the others), so that its draws, or an evaluation's greedy ones,
serve as targets: the flat head then answers with one softmax in place of two.
Masters are fp32, the GEMM operands bf16 copies that the optimizer refreshes.
state_bits=32 holds the moments in full: 0.1 MB more for these 17,000 parameters,
and no walk of the 8-bit rounding.
"""
import torch

from . import gemm as G
from ._lib import check, launch_stream, library, resolve_device
from .adamw import AdamW
from .conv_policy import WIDTH
from .layer_norm import layer_norm, layer_norm_backward
from .token_logprob import token_logprob, token_logprob_backward

F32 = torch.float32
JOINT, PITCH = 28, 32  # joint actions; logits of a row with their padding


def joint_legal(legal):
    """The 28 joint actions' legal bits (int32 [n]) from the environments' 12 (int16
    [n]): MOVE towards passable directions; ATTACK in those and at the nearest,
    with an adjacent visible monster; WAIT, REST, DESCEND."""
    bits = legal.to(torch.int32) & 0xfff
    walk, near = bits & 0xff, (bits >> 10) & 1
    return walk | near * (walk << 9 | 1 << 17) | ((bits >> 8) & 3) << 18 | ((bits >> 11) & 1) << 20


class JointHead:
    def __init__(self, device='cuda', seed=0, lr=3e-4, weight_decay=0.01, max_grad_norm=0.5, ent_coef=0.0, state_bits=8):
        self.device = dev = resolve_device(device)
        g = torch.Generator(device='cpu').manual_seed(seed)
        w = torch.zeros(PITCH, WIDTH, dtype=F32)
        w[:JOINT] = torch.randn(JOINT, WIDTH, generator=g, dtype=F32) / WIDTH ** 0.5
        f32 = dict(dtype=F32, device=dev)
        self.params = {'w': w.to(dev), 'b': torch.zeros(PITCH, **f32), 'norm_w': torch.ones(WIDTH, **f32),
                       'norm_b': torch.zeros(WIDTH, **f32)}
        self.grads = {k: torch.zeros_like(p) for k, p in self.params.items()}
        self.w = self.params['w'].to(torch.bfloat16)
        self.ent_coef = ent_coef
        self.optimizer = AdamW(self.params.values(), self.grads.values(), lr=lr, state_bits=state_bits,
                               weight_decay=[weight_decay, 0.0, 0.0, 0.0], max_norm=max_grad_norm,
                               copies=[self.w, None, None, None], seed=seed)
        self.lib = library()

    def forward(self, h, joint, legal, top=0):
        """(TokenLogprob of the actions `joint`, what the backward pass needs)."""
        y, mean, rstd = layer_norm(h, self.params['norm_w'], self.params['norm_b'])
        logits = G.gemm(y, self.w, bias=self.params['b'])[:, :JOINT]
        bits = joint_legal(legal)
        r = token_logprob(logits, joint, legal=bits, top=top)
        return r, (h, joint, y, mean, rstd, logits, bits)

    def alternatives(self, h, legal, top=4):
        """The `top` likeliest legal joint actions of each row (-1 where there are fewer) and their log-probabilities."""
        none = torch.full((h.shape[0],), -1, dtype=torch.int64, device=self.device)
        r, _ = self.forward(h, none, legal, top)
        return r.top_tokens, r.top_logp

    def backward(self, r, saved, dlogp, dentropy):
        """Fills self.grads; returns the gradient of the features (bf16)."""
        h, joint, y, mean, rstd, logits, bits = saved
        n, g = h.shape[0], self.grads
        dl = torch.zeros((n, PITCH), dtype=torch.bfloat16, device=self.device)
        token_logprob_backward(logits, joint, r.stats, r.entropy, dlogp, dentropy, legal=bits, out=dl[:, :JOINT])
        slabs = torch.empty((G.splits_for(n, 8), PITCH, WIDTH), dtype=F32, device=self.device)
        G.gemm_ex(dl, y, a_kn=True, b_kn=True, out_f32=slabs, splits=slabs.shape[0])
        check(self.lib.d1_reduce_slabs(slabs.data_ptr(), slabs.shape[0], PITCH * WIDTH, g['w'].data_ptr(),
                                       launch_stream(self.device)), 'd1_reduce_slabs')
        torch.sum(dl, 0, dtype=F32, out=g['b'])
        dh, dw, db = layer_norm_backward(G.gemm_bkn(dl, self.w), h, mean, rstd, self.params['norm_w'])
        g['norm_w'].copy_(dw)
        g['norm_b'].copy_(db)
        return dh

    def update(self, h, joint, legal):
        """One step on rows h (bf16 [n, 512]) with the actions `joint` (int64 [n], -1:
        none) taken where `legal` (the environments' bits) held. Returns the rows'
        log-probabilities and entropies before the step, on the device."""
        n = h.shape[0]
        r, saved = self.forward(h, joint, legal)
        dlogp = torch.full((n,), -1.0 / n, dtype=F32, device=self.device)
        dentropy = torch.full((n,), -self.ent_coef / n, dtype=F32, device=self.device) if self.ent_coef else None
        self.backward(r, saved, dlogp, dentropy)
        self.optimizer.step()
        return r.logp, r.entropy
