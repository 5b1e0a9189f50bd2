"""The policy/value network that sits on the other side of the `actor` batch (cfg 5).

PyTorch-ROCm plumbing, not part of the hot path: the shape of the reference's `Model_PolicyValue`
(go/df_model2.py:28-94: a 3x3 conv + BatchNorm + LeakyReLU(0.1) stem, `num_block` residual blocks of two
such layers at `dim` channels, 1x1 heads, softmax policy over the 361 points, tanh value) with the
reference's parameter names (`init_conv`, `conv_lower<i>`, `conv_upper<i>`, `pi_final_conv`,
`value_final_conv`, `pi_linear`, `value_linear1`, `value_linear2`), so a state dict saved by the
reference loads here.  Random-initialised when no checkpoint is given (none exists in this repo).

``norm="group"`` puts group norm in place of BatchNorm: a position's outputs do not depend on the rest of its batch
(selfplay batches of changing size, single positions), and norm, residual sum and activation are one kernel
(``policy_ops.group_norm_act``; the net runs channels last; ``groups`` divides ``dim``, and a head of two channels or one
has gcd(groups, its channels)).  ``dropout=p`` drops inside the residual blocks while the net is in training mode
(``policy_ops.dropout``; call ``next_step()`` after every optimizer step).
"""
import math

import torch
import torch.nn as nn

from . import policy_ops


class PolicyValueNet(nn.Module):
    def __init__(self, num_planes=25, dim=128, num_block=20, board_size=19, leaky_relu=True, bn=True, norm="batch", groups=8,
                 dropout=0.0, dropout_seed=0):
        super().__init__()
        if norm not in ("batch", "group"):
            raise ValueError("norm must be batch or group (got %r)" % (norm,))
        if norm == "group" and (not isinstance(groups, int) or groups < 1 or dim % groups):
            raise ValueError("groups must be a positive integer that divides the %d channels (got %r)" % (dim, groups))
        self.board_size, self.dim, self.num_block, self.bn = board_size, dim, num_block, bn
        self.groups = groups if norm == "group" else 0
        self.act = "leaky_relu" if leaky_relu else "relu"
        self.relu = nn.LeakyReLU(0.1) if leaky_relu else nn.ReLU()
        self.dropout = dropout
        if dropout:
            self.dropout_state = policy_ops.DropoutState(dropout_seed)
        self.init_conv = self._layer(num_planes, dim)
        for i in range(num_block):
            setattr(self, "conv_lower%d" % i, self._layer(dim, dim))
            setattr(self, "conv_upper%d" % i, self._layer(dim, dim, relu=False))
        self.pi_final_conv = self._layer(dim, 2, kernel=1)
        self.value_final_conv = self._layer(dim, 1, kernel=1)
        d = board_size * board_size
        self.pi_linear = nn.Linear(2 * d, d)
        self.value_linear1 = nn.Linear(d, 256)
        self.value_linear2 = nn.Linear(256, 1)

    def _layer(self, cin, cout, kernel=3, relu=True):
        mods = [nn.Conv2d(cin, cout, kernel, padding=kernel // 2)]
        if self.groups:
            return nn.Sequential(*mods, policy_ops.GroupNormAct(math.gcd(self.groups, cout), cout, act=self.act if relu else "none"))
        if self.bn:
            mods.append(nn.BatchNorm2d(cout))
        if relu:
            mods.append(self.relu)
        return nn.Sequential(*mods)

    def _apply_layer(self, layer, s, residual=None):
        if not self.groups:
            return layer(s)
        conv, norm = layer
        return norm(conv(s).contiguous(memory_format=torch.channels_last), residual)

    def _block(self, i, s):
        lower, upper = getattr(self, "conv_lower%d" % i), getattr(self, "conv_upper%d" % i)
        t = self._apply_layer(lower, s)
        if self.dropout and self.training:
            t = policy_ops.dropout(t, self.dropout, self.dropout_state.rng, site=i)
        if self.groups:                              # norm, sum and activation in one
            conv, norm = upper
            return policy_ops.group_norm_act(conv(t).contiguous(memory_format=torch.channels_last), norm.num_groups, norm.weight,
                                             norm.bias, norm.eps, self.act, residual=s)
        return self.relu(upper(t) + s)

    def forward(self, x, legal=None, temperature=1.0):
        """x: the batch (anything answering ["s"]) or the planes tensor [B, 25, 19, 19].  legal: the environment's mask [B, 361]:
        pi is then taken over the legal points (a row without one gives zeros, for which the environment falls back to its
        uniform policy).  temperature: a number, or a float32 tensor [B]; pi's logits are divided by it."""
        s = x if torch.is_tensor(x) else x["s"]
        s = s.to(self.pi_linear.weight.dtype)
        if self.groups:
            s = s.contiguous(memory_format=torch.channels_last)
        s = self._apply_layer(self.init_conv, s)
        for i in range(self.num_block):
            s = self._block(i, s)
        d = self.board_size * self.board_size
        logits = self.pi_linear(self._apply_layer(self.pi_final_conv, s).reshape(-1, 2 * d))
        if legal is None and not torch.is_tensor(temperature) and temperature == 1.0:
            pi = torch.softmax(logits, dim=1)
        else:
            pi = policy_ops.policy_logits(logits, legal=legal, temperature=temperature, out="probs", dtype=torch.float32)
        v = self.relu(self.value_linear1(self._apply_layer(self.value_final_conv, s).reshape(-1, d)))
        return dict(pi=pi, V=torch.tanh(self.value_linear2(v)))

    def next_step(self):
        """New dropout masks from here on: once per training step, after its backward pass."""
        if self.dropout:
            self.dropout_state.advance()


def make_actor(net, mask_policy=False, temperature=1.0):
    """The callback of the `actor` collector: what Evaluator.actor replies without a sampler
    (rlpytorch/trainer/trainer.py:57-91: pi, and V) -- the environment samples the move from pi over
    the legal points on the device.  mask_policy: the net's pi is taken over the batch's `legal` points already (the
    key has to be among the batch's inputs, go_loader's --legal_mask), with the given temperature."""
    def actor(batch):
        b = batch.hist(0)
        with torch.no_grad():
            out = net(b, b["legal"] if mask_policy else None, temperature)
        return dict(pi=out["pi"].float(), V=out["V"].float().view(-1))
    return actor
