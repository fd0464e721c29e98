"""A layer of latent attention through its three uses: training steps on whole
sequences (expanded form, autograd), a prompt into the paged cache, and tokens
one at a time out of it (absorbed form).

    python examples/latent_layer.py

The same weights and tokens have to give the same outputs in all three, up to
bfloat16 rounding; the script checks that and prints what it measured.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "atomic_ai_hybrid-v0.1_amd"))
from atomic_ops import latent  # noqa: E402


class LatentLayer(torch.nn.Module):
    def __init__(self, width=512, heads=6, dn=128, dr=64, dv=128, dc=512, positions=4096):
        super().__init__()
        self.heads, self.dn, self.dr, self.dv, self.dc = heads, dn, dr, dv, dc
        self.scale = (dn + dr) ** -0.5
        w = lambda o, i: torch.nn.Parameter((torch.randn(o, i) * i ** -0.5).to(torch.bfloat16))
        self.w_q, self.w_down = w(heads * (dn + dr), width), w(dc + dr, width)
        self.w_kv, self.w_o = w(heads * (dn + dv), dc), w(width, heads * dv)
        a = torch.arange(positions)[:, None] * 1e4 ** (-torch.arange(0, dr, 2) / dr)
        self.register_buffer("cos", a.cos())
        self.register_buffer("sin", a.sin())

    def _rotate(self, x, t0=0):
        """Differentiable rotation of [.., T, (H,) dr]: pairs (i, i + dr / 2), as ``latent.append`` does it."""
        T = x.shape[1]
        shape = (T,) + (1,) * (x.dim() - 3) + (self.dr // 2,)
        c, s = self.cos[t0:t0 + T].view(shape), self.sin[t0:t0 + T].view(shape)
        a, b = x.float().chunk(2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1).to(x.dtype)

    def forward(self, x, lens=None):
        """Whole sequences [B, T, width] (``lens`` int32 [B] of them real), differentiable."""
        B, T, _ = x.shape
        q = (x @ self.w_q.t()).view(B, T, self.heads, -1)
        c, k_pe = (x @ self.w_down.t()).split((self.dc, self.dr), -1)
        kv = (c @ self.w_kv.t()).view(B, T, self.heads, -1)
        q = torch.cat((q[..., :self.dn], self._rotate(q[..., self.dn:])), -1)
        o = latent.attention(q, kv, self._rotate(k_pe), self.scale, q_lens=lens, kv_lens=lens)
        return o.flatten(2) @ self.w_o.t()

    @torch.no_grad()
    def prompt(self, x, cache, slots):
        """One sequence [T, width] into the cache rows ``slots`` [T]; its outputs."""
        T = x.shape[0]
        q = (x @ self.w_q.t()).view(T, self.heads, -1)
        down = x @ self.w_down.t()
        pos = torch.arange(T, dtype=torch.int32, device=x.device)
        k_pe, q = latent.append(cache, down[:, :self.dc], down[:, self.dc:], slots, pos, self.cos, self.sin, q=q)
        kv = (down[:, :self.dc] @ self.w_kv.t()).view(T, self.heads, -1)
        o, _ = latent.forward(q[None], kv[None], k_pe[None], self.scale)
        return o[0].flatten(1) @ self.w_o.t()

    @torch.no_grad()
    def step(self, x, cache, table, lens, slots):
        """The next token of each sequence [B, width]; ``lens`` count it in, ``slots`` are its cache rows."""
        B = x.shape[0]
        q = (x @ self.w_q.t()).view(B, 1, self.heads, -1)
        down = x @ self.w_down.t()
        latent.append(cache, down[:, :self.dc], down[:, self.dc:], slots, lens - 1, self.cos, self.sin)
        w_kv = self.w_kv.view(self.heads, self.dn + self.dv, self.dc)
        o = latent.decode(q, w_kv, cache, table, lens, self.scale, cos=self.cos, sin=self.sin)
        return o.flatten(1) @ self.w_o.t()


def main(B=3, T=200, prompt=150, page=64, steps=5):
    torch.manual_seed(0)
    layer = LatentLayer().cuda()
    x = torch.randn(B, T, 512, device="cuda").to(torch.bfloat16)
    target = torch.randn(B, T, 512, device="cuda")
    opt = torch.optim.SGD(layer.parameters(), lr=20.0)
    losses = []
    for _ in range(steps):
        loss = (layer(x).float() - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    print("training loss", " ".join(f"{v:.4f}" for v in losses))
    assert losses[-1] < losses[0]

    want = layer(x).detach().float()
    per = -(-T // page)
    cache = torch.zeros(B * per, page, layer.dc + layer.dr, dtype=torch.bfloat16, device="cuda")
    table = torch.randperm(B * per, device="cuda").view(B, per).to(torch.int32)
    slot = lambda b, t: table[b, t // page].long() * page + t % page
    at = torch.arange(prompt, device="cuda")
    got = torch.empty_like(want)
    for b in range(B):
        got[b, :prompt] = layer.prompt(x[b, :prompt], cache, slot(b, at))
    rows = torch.arange(B, device="cuda")
    for t in range(prompt, T):
        lens = torch.full((B,), t + 1, dtype=torch.int32, device="cuda")
        now = torch.full((B,), t, device="cuda")
        got[:, t] = layer.step(x[:, t], cache, table, lens, slot(rows, now))
    off = lambda a, b: ((a - b).norm() / b.norm()).item()
    p, s = off(got[:, :prompt], want[:, :prompt]), off(got[:, prompt:], want[:, prompt:])
    print(f"against the training form: prompt {p:.4f}, tokens {s:.4f} of the norm")
    assert max(p, s) < 0.02
    return losses, p, s


if __name__ == "__main__":
    main()
