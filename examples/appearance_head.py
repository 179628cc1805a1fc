"""A learned appearance on top of the splats: their colours shift with the lighting of each view, and a gated feed-forward head
learns how, from the rasterizer's own colour gradients.

    python examples/appearance_head.py [--splats 4096] [--steps 60]

Every splat is a row: random Fourier features of its position beside a code of the view. The head (nn.FeedForward) turns a row
into an offset of the splat's DC colour. A step puts one view's features through dropout (nn.Dropout) and the head, whose output
is dropped out in its own epilogue, renders with the shifted colours, takes the photometric loss and its gradient, and hands the
colours' gradients back to the head; the weights follow by Adam in single precision. At the end the weights are rounded to 8 bits
(nn.QuantizeRows) and the views are rendered from the 8-bit head (nn.I8FeedForward).
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np

from b2ctrain_amd import _native, nn
from b2ctrain_amd import scenes as S

WIDTH, HIDDEN, CODE = 64, 256, 8


def bf16(x):
    """float32 values as bfloat16 bits, to nearest even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


class Mat:
    """A bfloat16 or single-precision matrix on the device, with its nn.Matrix."""

    def __init__(self, x, dtype=nn.BF16):
        self.shape, self.dtype = x.shape, dtype
        self.put(x)

    def put(self, x):
        host = bf16(x) if self.dtype == nn.BF16 else np.ascontiguousarray(x, np.int8 if self.dtype == nn.I8 else np.float32)
        self.dev = _native.DeviceArray(host)
        self.matrix = nn.Matrix(self.dev.ptr, *self.shape, self.shape[1], self.dtype, keep=self.dev)

    def get(self):
        if self.dtype == nn.BF16:
            return from_bf16(self.dev.download(np.uint16, self.shape))
        return self.dev.download(np.int8 if self.dtype == nn.I8 else np.float32, self.shape)


def room(n):
    return _native.DeviceArray(np.zeros(n, np.uint8))


class Adam:
    def __init__(self, arrays, lr):
        self.p, self.lr, self.t = arrays, lr, 0
        self.m, self.v = [np.zeros_like(a) for a in arrays], [np.zeros_like(a) for a in arrays]

    def step(self, grads):
        self.t += 1
        for p, m, v, g in zip(self.p, self.m, self.v, grads):
            m += 0.1 * (g - m)
            v += 0.001 * (g * g - v)
            p -= self.lr * (m / (1 - 0.9 ** self.t)) / (np.sqrt(v / (1 - 0.999 ** self.t)) + 1e-8)


class Lit:
    """A cloud whose views are lit by different colours, and the renderer of each shifted cloud."""

    def __init__(self, splats, views, seed):
        g = np.random.default_rng(seed)
        self.scene = S.config2(n=splats)
        self.scene.sh[:, 1:] = 0
        self.base = self.scene.sh[:, 0].copy()
        W = H = 128
        c = self.scene.cam
        self.scene.cam = S.Camera(W, H, c.fx * W / c.width, c.fy * H / c.height, W / 2, H / 2, c.R, c.t)
        self.scene.gt = np.zeros(W * H, np.uint32)
        self.r = _native.Renderer(self.scene, W, H)
        pos = self.scene.pos_op[:, :3]
        # what a view's light does to a splat's colour: a smooth function of where it is
        lights = g.standard_normal((views, 3, 3)) * 0.8
        self.truth = [np.tanh(pos @ lights[v]) * 0.6 for v in range(views)]
        self.targets = []
        for v in range(views):
            self.shift(self.truth[v])
            self.r.forward()
            rgba = np.clip(self.r.read("out_rgba"), 0, 1)
            self.targets.append(S._pack_rgba(rgba[:, 0], rgba[:, 1], rgba[:, 2], np.ones(W * H)))
        waves = g.standard_normal((3, (WIDTH - CODE) // 2)) * 1.5
        codes = g.standard_normal((views, CODE))
        f = np.concatenate([np.sin(pos @ waves), np.cos(pos @ waves)], axis=1)
        self.features = [np.concatenate([f, np.tile(codes[v], (splats, 1))], axis=1).astype(np.float32) for v in range(views)]

    def shift(self, offset):
        self.scene.sh[:, 0] = self.base + offset
        self.r.upload(self.scene)

    def loss(self, v, offset, grad=False):
        """The photometric loss of view v with the colours shifted, and its gradient by the offsets."""
        self.shift(offset)
        self.r.set_target(self.targets[v])
        self.r.forward()
        scale = 3.0 * self.r.W * self.r.H if grad else 1.0
        loss = self.r.loss(grad_scale=scale) - self.scene.ssim_w  # 0 for the target itself, whose SSIM is 1
        if not grad:
            return loss, None
        self.r.backward(grad_scale=scale)
        self.r.vjp()
        return loss, self.r.read("grads")[:, 11:14]


def run(splats=4096, steps=60, views=3, p=0.05, seed=1, say=print):
    g = np.random.default_rng(seed)
    lit = Lit(splats, views, seed)
    draw = lambda o, i, k: (g.standard_normal((o, i)) * k / np.sqrt(i)).astype(np.float32)  # noqa: E731
    params = [draw(HIDDEN, WIDTH, 1.0), draw(HIDDEN, WIDTH, 1.0), draw(WIDTH, HIDDEN, 0.05)]
    w = [Mat(a) for a in params]
    adam = Adam(params, 4e-3)
    features = [Mat(f) for f in lit.features]
    x, y, dy = Mat(np.zeros((splats, WIDTH))), Mat(np.zeros((splats, WIDTH))), Mat(np.zeros((splats, WIDTH)))
    grads = [Mat(np.zeros(a.shape), nn.F32) for a in params]

    def losses(offsets):
        return [lit.loss(v, offsets(v))[0] for v in range(views)]

    start = losses(lambda v: 0)
    for step in range(steps):
        v = step % views
        for m, a in zip(w, params):
            m.put(a)
        nn.Dropout(features[v].matrix, x.matrix, p, seed, 2 * step).run()
        head = nn.FeedForward(x.matrix, w[0].matrix, w[1].matrix, w[2].matrix, y.matrix, p=p, seed=seed, stream_id=2 * step + 1,
                              train=True, room=room)
        head.forward()
        loss, d = lit.loss(v, y.get()[:, :3], grad=True)
        d = np.pad(d, ((0, 0), (0, WIDTH - 3)))
        dy.put(d / max(np.abs(d).max(), 1e-20))  # Adam does not see the scale
        head.gradients(dy.matrix, dw_gate=grads[0].matrix, dw_up=grads[1].matrix, dw_down=grads[2].matrix, room=room)
        head.backward()
        adam.step([m.get() for m in grads])
        if step % 10 == 0 or step + 1 == steps:
            say(f"step {step}: view {v}, loss {loss:.4f}")
    for m, a in zip(w, params):
        m.put(a)

    q = []
    for m in w:
        q8, s = Mat(np.zeros(m.shape), nn.I8), Mat(np.zeros((m.shape[0], 1)), nn.F32)
        nn.QuantizeRows(m.matrix, q8.matrix, s.matrix).run()
        q.append((q8, s))

    def answer(v, eight):
        if eight:
            (g8, gs), (u8, us), (d8, ds) = q
            nn.I8FeedForward(features[v].matrix, g8.matrix, gs.matrix, u8.matrix, us.matrix, d8.matrix, ds.matrix, y.matrix, room=room).run()
        else:
            nn.FeedForward(features[v].matrix, w[0].matrix, w[1].matrix, w[2].matrix, y.matrix, room=room).forward()
        return y.get()[:, :3]

    full, eight = losses(lambda v: answer(v, False)), losses(lambda v: answer(v, True))
    for v in range(views):
        say(f"view {v}: loss {start[v]:.4f} without the head, {full[v]:.4f} with it, {eight[v]:.4f} with it in 8 bits")
    lit.r.close()
    return start, full, eight


if __name__ == "__main__":
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--splats", type=int, default=4096)
    a.add_argument("--steps", type=int, default=60)
    args = a.parse_args()
    run(args.splats, args.steps)
