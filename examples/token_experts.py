"""A token classifier trained through the library's reverse sweeps.

    ids -> embed -> layer_norm -> rows grouped by expert -> expert_mm -> gelu
    (its input kept on the 8-bit tape) -> expert_mm -> rows back in order,
    added to the embedding -> layer_norm -> mlp2_ce (tanh layer, softmax
    cross-entropy) per position

Positions are routed by a fixed table (id modulo the number of experts); the
grouping and its inverse are gathers by an index list, which is what embed
does with any array, and embed_b of one is the gather by the other. The head
is the Float32 MLP sweep, everything before it runs in the chosen type with
Float32 parameter gradients and a Float32 copy of the parameters.

Run on a GPU: python examples/token_experts.py [--dtype bf16] [--steps 200]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "stade.jl_b200"))
import stadeb200 as sb  # noqa: E402

EPS = 1e-5


class TokenExperts:
    """Parameters (Float32 masters in self.p), gradients (self.g) and the
    buffers of one batch size."""

    def __init__(self, n_s, n_v, n_d, n_e, n_f, n_h, n_o, dtype=torch.bfloat16, act="gelu", seed=0):
        self.size = (n_s, n_v, n_d, n_e, n_f, n_h, n_o)
        self.dtype, self.act = dtype, act
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=g) * scale).cuda()

        self.p = {"table": normal(n_v, n_d, scale=1 / math.sqrt(n_d)),
                  "norm_w": torch.ones(n_d).cuda(), "norm_b": torch.zeros(n_d).cuda(),
                  "up": normal(n_e, n_d, n_f, scale=1 / math.sqrt(n_d)),
                  "down": normal(n_e, n_f, n_d, scale=0.5 / math.sqrt(n_f)),
                  "out_w": torch.ones(n_d).cuda(), "out_b": torch.zeros(n_d).cuda(),
                  "w1": normal(n_d, n_h, scale=1 / math.sqrt(n_d)), "b1": torch.zeros(n_h).cuda(),
                  "w2": normal(n_h, n_o, scale=1 / math.sqrt(n_h)), "b2": torch.zeros(n_o).cuda()}
        self.g = {k: torch.zeros_like(v) for k, v in self.p.items()}

        def rows(n, t=dtype):
            return torch.zeros(n_s, n, dtype=t, device="cuda")

        f = torch.float32
        # forward values and, where a name ends in b, their adjoints
        self.b = {k: rows(n_d) for k in ("emb", "embb", "norm", "normb", "xg", "xgb", "yg", "ygb",
                                         "y", "yb", "res", "resb", "out", "outb")}
        self.b |= {k: rows(n_f) for k in ("up", "upb", "hid", "hidb")}
        self.b |= {"x": rows(n_d, f), "xb": rows(n_d, f), "h": rows(n_h, f), "hb": rows(n_h, f)}
        self.b |= {k: rows(n_o, f) for k in ("t", "tb", "z", "zb", "p", "pb")}
        self.stats = [torch.empty(n_s, device="cuda") for _ in range(4)]
        self.q, self.e = sb.initstacks_tape8_cuda(n_s, n_f)
        self.loss, self.lossb = torch.zeros(1, device="cuda"), torch.full((1,), 1 / n_s, device="cuda")

    def route(self, ids):
        """(order, place, bounds): the positions grouped by expert, where each
        position went, and the groups' bounds; all on the device."""
        n_e = self.size[3]
        expert = ids % n_e
        order = torch.argsort(expert, stable=True)
        place = torch.empty_like(order)
        place[order] = torch.arange(len(ids), device=ids.device)
        bounds = torch.zeros(n_e + 1, dtype=torch.int64, device=ids.device)
        bounds[1:] = torch.cumsum(torch.bincount(expert, minlength=n_e), 0)
        return order, place, bounds

    def gradient(self, ids, target):
        """Mean loss of the batch (a device scalar) and, in self.g, its gradient.
        ids: int64 positions; target: n_s x n_o one-hot rows."""
        n_s, n_v, n_d, n_e, n_f, n_h, n_o = self.size
        b, p, g, dt = self.b, self.p, self.g, self.dtype
        m1, r1, m2, r2 = self.stats
        table, up, down = (p[k].to(dt) for k in ("table", "up", "down"))
        order, place, bounds = self.route(ids)

        sb.embed_cuda(table, ids, b["emb"], math.sqrt(n_d), n_s, n_v, n_d)
        sb.layer_norm_cuda(b["emb"], p["norm_w"], p["norm_b"], b["norm"], m1, r1, EPS, n_s, n_d)
        sb.embed_cuda(b["norm"], order, b["xg"], 1.0, n_s, n_s, n_d)
        sb.expert_mm_cuda(b["xg"], up, b["up"], bounds, n_s, n_e, n_d, n_f)
        sb.act_tape8_cuda(self.act, b["up"], b["hid"], self.q, self.e, n_s, n_f)
        sb.expert_mm_cuda(b["hid"], down, b["yg"], bounds, n_s, n_e, n_f, n_d)
        sb.embed_cuda(b["yg"], place, b["y"], 1.0, n_s, n_s, n_d)
        torch.add(b["emb"], b["y"], out=b["res"])
        sb.layer_norm_cuda(b["res"], p["out_w"], p["out_b"], b["out"], m2, r2, EPS, n_s, n_d)

        # the head's sweep adds to its adjoints and leaves the intermediate ones at zero
        b["x"].copy_(b["out"])
        b["t"].copy_(target)
        self.loss.zero_()
        for t in (b["xb"], b["tb"], g["w1"], g["b1"], g["w2"], g["b2"]):
            t.zero_()
        sb.mlp2_ce_b_cuda(self.loss, self.lossb, b["x"], b["xb"], b["t"], b["tb"], p["w1"], g["w1"],
                          p["b1"], g["b1"], p["w2"], g["w2"], p["b2"], g["b2"], b["h"], b["hb"],
                          b["z"], b["zb"], b["p"], b["pb"], n_s, n_d, n_h, n_o)

        # in reverse; the seeds are overwritten by the next step, so none is cleared
        new = dict(accumulate=False, consume=False)
        b["outb"].copy_(b["xb"])
        sb.layer_norm_b_cuda(b["res"], b["resb"], p["out_w"], g["out_w"], g["out_b"], b["outb"], m2,
                             r2, n_s, n_d, **new)
        sb.embed_cuda(b["resb"], order, b["ygb"], 1.0, n_s, n_s, n_d)      # place's inverse
        sb.expert_mm_b_cuda(b["hid"], b["hidb"], down, g["down"], b["ygb"], bounds, n_s, n_e, n_f,
                            n_d, **new)
        sb.act_tape8_b_cuda(self.act, b["upb"], b["hidb"], self.q, self.e, n_s, n_f, **new)
        sb.expert_mm_b_cuda(b["xg"], b["xgb"], up, g["up"], b["upb"], bounds, n_s, n_e, n_d, n_f,
                            **new)
        sb.embed_cuda(b["xgb"], place, b["normb"], 1.0, n_s, n_s, n_d)     # order's inverse
        b["embb"].copy_(b["resb"])
        sb.layer_norm_b_cuda(b["emb"], b["embb"], p["norm_w"], g["norm_w"].zero_(),
                             g["norm_b"].zero_(), b["normb"], m1, r1, n_s, n_d)   # adds to embb
        sb.embed_b_cuda(g["table"], ids, b["embb"], math.sqrt(n_d), n_s, n_v, n_d, **new)
        # the sweep sums the loss over positions; its seed makes the gradients a mean's
        return self.loss / n_s

    def step(self, ids, target, rate):
        """One step of gradient descent; returns the loss before it."""
        loss = self.gradient(ids, target)
        for k, v in self.p.items():
            v.add_(self.g[k], alpha=-rate)
        return loss


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--dtype", choices=["f32", "bf16", "f16"], default="bf16")
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--positions", type=int, default=4096)
    a = ap.parse_args()
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[a.dtype]
    n_v, n_o = 5000, 10
    model = TokenExperts(a.positions, n_v, 256, 8, 512, 128, n_o, dt)
    g = torch.Generator(device="cuda").manual_seed(1)
    labels = torch.randint(0, n_o, (n_v,), generator=g, device="cuda")   # each id's class
    for i in range(a.steps):
        ids = torch.randint(0, n_v, (a.positions,), generator=g, device="cuda")
        target = torch.nn.functional.one_hot(labels[ids], n_o)
        loss = model.step(ids, target, rate=1.0)
        if i % 20 == 0 or i + 1 == a.steps:
            print(f"step {i:4d}  loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
