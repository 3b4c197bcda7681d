"""One training step of the matching network (the network of reference ffn.py:225-265; its loss and optimiser are those of Keras:
binary cross-entropy, Adam, global_clipnorm).  FFN.compile / FFN.train_on_batch are the entry points.

The dense layers and their gradients are grouped products (grouped.py): the first layer is one group of all rows, the second two -- the reference
cells with the upper half of its weights, the target cells with the lower half -- so the rows of both halves go through one launch and the
concatenated 1024-column table is never built.  The gradients of all tensors are clipped together (gradients.py).  Batch normalisation, LeakyReLU, the
loss and the update are element-wise torch expressions.  Keras' semantics: BN1 is called once for each half (its own statistics each, the moving
averages updated twice), variances are biased, momentum 0.99, epsilon 1e-3; Adam with epsilon 1e-7.  No Keras is available to pin them to."""
from __future__ import annotations

import numpy as np

from . import _dev
from .arch import FFN_FEAT
from .gradients import clip_by_global_norm
from .grouped import product, product_grad

SLOPE, EPS, MOMENTUM = 0.3, 1e-3, 0.99
TRAINED = ("w1", "gamma1", "beta1", "w2", "gamma2", "beta2", "w3", "b3")


class FFNTraining:
    """The network's weights on the GPU, in 32 bits, with Adam's moments"""

    def __init__(self, weights: dict, device, learning_rate: float = 1e-3, beta_1: float = 0.9, beta_2: float = 0.999, epsilon: float = 1e-7,
                 global_clipnorm: float | None = None):
        t = _dev.torch()
        if global_clipnorm is not None and not 0 < global_clipnorm < float("inf"):
            raise ValueError(f"global_clipnorm must be positive and finite, got {global_clipnorm}")
        self.rate, self.b1, self.b2, self.eps, self.clip = float(learning_rate), float(beta_1), float(beta_2), float(epsilon), global_clipnorm
        up = lambda a, shape: t.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=np.float32)).reshape(shape)).to(device)
        hid = np.asarray(weights["w3"]).size
        first = {"w1": up(weights["w1"], (1, FFN_FEAT, hid)), "gamma1": up(weights["bn1"]["gamma"], hid), "beta1": up(weights["bn1"]["beta"], hid),
                 "w2": up(weights["w2"], (2, hid, hid)), "gamma2": up(weights["bn2"]["gamma"], hid), "beta2": up(weights["bn2"]["beta"], hid),
                 "w3": up(weights["w3"], (1, hid, 1)), "b3": up(weights["b3"], 1)}
        # one buffer for all weights, views for each: the update is a handful of launches
        self.flat = t.cat([first[k].reshape(-1) for k in TRAINED])
        self.grad, self.m, self.v = t.zeros_like(self.flat), t.zeros_like(self.flat), t.zeros_like(self.flat)
        views = lambda buf: dict(zip(TRAINED, (p.view(first[k].shape) for k, p in zip(TRAINED, t.split(buf, [first[k].numel() for k in TRAINED])))))
        self.w, self.g = views(self.flat), views(self.grad)
        self.moving = {k: up(weights[b][n], hid).clone() for k, b, n in (("mean1", "bn1", "mean"), ("var1", "bn1", "var"), ("mean2", "bn2", "mean"), ("var2", "bn2", "var"))}
        self.steps, self.offsets = 0, {}

    @staticmethod
    def _normalise(h, gamma, beta):
        """h [parts][rows][c]: batch normalisation with each part's own statistics, then LeakyReLU -> (activations, what the backward pass needs)"""
        mean = h.mean(1, keepdim=True)
        var = (h - mean).square().mean(1, keepdim=True)
        rstd = (var + EPS).rsqrt()
        hat = (h - mean) * rstd
        z = hat * gamma + beta
        return z.where(z >= 0, SLOPE * z), (hat, rstd, z >= 0, mean[:, 0], var[:, 0])

    @staticmethod
    def _normalise_grad(dy, saved, gamma):
        hat, rstd, up, _, _ = saved
        dz = dy.where(up, SLOPE * dy)
        dbeta, dgamma = dz.sum(1, keepdim=True), (dz * hat).sum(1, keepdim=True)
        dh = gamma * rstd * (dz - (dbeta + hat * dgamma) / dy.shape[1])
        return dh, dgamma.sum((0, 1)), dbeta.sum((0, 1))

    def gradients(self, x, y):
        """x [rows][122], y [rows] on the GPU -> (loss, {name: gradient}, the batch's statistics)"""
        t = _dev.torch()
        rows, hid = x.shape[0], self.w["w3"].shape[1]
        halves = x.view(rows, 2, FFN_FEAT).transpose(0, 1).reshape(2 * rows, FFN_FEAT)
        if rows not in self.offsets:                                  # one group of all rows, the two halves, the rows of the pairs
            self.offsets = {rows: [t.tensor(o, dtype=t.int32).to(x.device) for o in ([0, 2 * rows], [0, rows, 2 * rows], [0, rows])]}
        one, two, last = self.offsets[rows]
        h1, s1 = self._normalise(product(halves, self.w["w1"], one).view(2, rows, hid), self.w["gamma1"], self.w["beta1"])
        h1 = h1.view(2 * rows, hid)
        pair = product(h1, self.w["w2"], two).view(2, rows, hid)
        h2, s2 = self._normalise((pair[0] + pair[1])[None], self.w["gamma2"], self.w["beta2"])
        h2 = h2[0]
        logit = product(h2, self.w["w3"], last)[:, 0] + self.w["b3"]
        loss = (t.nn.functional.softplus(logit) - y * logit).mean()
        g = {}
        d = ((t.sigmoid(logit) - y) / rows)[:, None]
        g["b3"] = d.sum().view(1)
        d, g["w3"] = product_grad(d, h2, self.w["w3"], last)
        d, g["gamma2"], g["beta2"] = self._normalise_grad(d[None], s2, self.w["gamma2"])
        d, g["w2"] = product_grad(d.expand(2, rows, hid).reshape(2 * rows, hid), h1, self.w["w2"], two)
        d, g["gamma1"], g["beta1"] = self._normalise_grad(d.view(2, rows, hid), s1, self.w["gamma1"])
        _, g["w1"] = product_grad(d.view(2 * rows, hid), halves, self.w["w1"], one, need_x=False)
        return loss, g, (s1[3], s1[4], s2[3], s2[4])

    def step(self, x, y):
        """One update from the rows x [rows][122] with labels y [rows] -> the loss before it, a scalar on the GPU"""
        loss, g, stats = self.gradients(x, y)
        grads = [g[k] for k in TRAINED]
        if self.clip is not None:
            clip_by_global_norm(grads, self.clip, out=[self.g[k].view(v.shape) for k, v in zip(TRAINED, grads)])
        else:
            for k, v in zip(TRAINED, grads):
                self.g[k].copy_(v)
        for name, batch in zip(("mean1", "var1", "mean2", "var2"), stats):
            for part in batch:                                        # once for each call of the layer
                self.moving[name].mul_(MOMENTUM).add_(part, alpha=1 - MOMENTUM)
        self.steps += 1
        self.m.mul_(self.b1).add_(self.grad, alpha=1 - self.b1)
        self.v.mul_(self.b2).addcmul_(self.grad, self.grad, value=1 - self.b2)
        rate = self.rate * (1 - self.b2 ** self.steps) ** 0.5 / (1 - self.b1 ** self.steps)
        self.flat.addcdiv_(self.m, self.v.sqrt().add_(self.eps), value=-rate)
        return loss

    def weights(self) -> dict:
        """The weights as numpy arrays, in the layout of FFN.set_weights_dict"""
        c = lambda a, *shape: a.detach().cpu().numpy().reshape(shape).copy()
        hid = self.w["w3"].shape[1]
        bn = lambda i: {"gamma": c(self.w[f"gamma{i}"], hid), "beta": c(self.w[f"beta{i}"], hid), "mean": c(self.moving[f"mean{i}"], hid), "var": c(self.moving[f"var{i}"], hid)}
        return {"w1": c(self.w["w1"], FFN_FEAT, hid), "bn1": bn(1), "w2": c(self.w["w2"], 2 * hid, hid), "bn2": bn(2), "w3": c(self.w["w3"], hid, 1), "b3": c(self.w["b3"], 1)}
