"""The two token mixers of a hybrid layer, run together as an executor uses them: a prompt in chunks, decoded
tokens one by one, and a tree of drafted tokens that is verified, accepted in part and rolled back.

Attention layer: q/k norm + RoPE + INT8 KV append in one launch, then attention over the cache (sliding window and
sinks). GDN layer: the gated delta rule, then its output's gated norm. Needs a B200 and the built library:

    python wzy-flash-serve_b200/example_mixers.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import wzyb200 as wz  # noqa: E402

F16, F32 = torch.float16, torch.float32


class AttentionMixer:
    """One attention layer's cache and calls. `ring` cells in HBM: 4096 pinned, the rest sliding."""

    def __init__(self, q_heads=16, kv_heads=2, head_dim=256, ring=32768, max_ctx=262144, window=8192, sinks=64,
                 chunk=4096, max_nodes=64, device="cuda"):
        self.qh, self.kvh, self.hd, self.window, self.sinks = q_heads, kv_heads, head_dim, window, sinks
        kvd = kv_heads * head_dim

        def planes(cells):
            return [torch.zeros(cells, w, dtype=t, device=device) for _ in range(2)
                    for w, t in ((kvd, torch.int8), (kvd // 64, torch.int16))]

        self.ring, self.draft_ring = planes(ring), planes(max_nodes)
        self.cache = wz.kv_cache(*self.ring, ring, max_ctx)
        self.drafts = wz.kv_cache(*self.draft_ring, max_nodes, max_nodes)
        self.q_gamma, self.k_gamma = (torch.zeros(head_dim, dtype=F16, device=device) for _ in range(2))
        self.cos, self.sin = (torch.empty(max_ctx, 32, device=device) for _ in range(2))
        wz.rope_table(self.cos, self.sin, max_ctx)
        need = max(wz.kv_attn_workspace_bytes(t, q_heads, kv_heads, head_dim) for t in (1, 2, 4, 8, 16, 32, 64, 256, chunk))
        self.ws = torch.empty(max(need, 16), dtype=torch.uint8, device=device)
        self.pos = torch.zeros(1, dtype=torch.int32, device=device)  # committed tokens, read by the kernels

    def forward(self, q, k, v):
        """Append T new tokens and attend: q [T, q_heads, d], k, v [T, kv_heads * d], fp16; k and q in place."""
        T = q.shape[0]
        heads = wz.head_tensor(q, self.q_gamma, self.qh, self.hd, self.qh * self.hd)
        wz.k_rope_kv_append(k, self.k_gamma, v, self.cos, self.sin, T, self.kvh, self.hd, self.cache, w_offset=1.0,
                            d_base_pos=self.pos, q=heads)
        out = torch.empty_like(q)
        ws = self.workspace(T)
        wz.kv_attn(q, out, self.cache, self.kvh, self.window, self.sinks, d_base_pos=self.pos, workspace=ws)
        self.pos += T
        return out

    def verify(self, q, k, v, mask, depth):
        """Attention of drafted nodes (q, k rotated at base + depth, fp32) without touching the cache."""
        n = q.shape[0]
        wz.kv_append_int8_f32(k, v, n, self.kvh, self.hd, self.drafts)
        out = torch.empty_like(q)
        wz.kv_tree_attn(q, out, self.cache, self.drafts, mask, self.kvh, self.window, depth, sinks=self.sinks,
                        d_base_pos=self.pos, workspace=self.workspace(n))
        return out

    def accept(self, k, v):
        """The accepted nodes' k, v (fp32, in order) become committed tokens."""
        n = k.shape[0]
        wz.kv_append_int8_f32(k.contiguous(), v.contiguous(), n, self.kvh, self.hd, self.cache, d_base_pos=self.pos)
        self.pos += n

    def workspace(self, T):
        need = wz.kv_attn_workspace_bytes(T, self.qh, self.kvh, self.hd)
        if need > self.ws.numel():
            self.ws = torch.empty(need, dtype=torch.uint8, device=self.ws.device)
        return self.ws


class GdnMixer:
    """One GDN layer's state and calls."""

    def __init__(self, k_heads=16, v_heads=32, head_dim=128, device="cuda"):
        self.kh, self.vh, self.hd = k_heads, v_heads, head_dim
        self.state = torch.zeros(v_heads, head_dim, head_dim, device=device)
        self.gamma = torch.ones(head_dim, dtype=F16, device=device)
        self.ws = torch.empty(16, dtype=torch.uint8, device=device)

    def forward(self, qkv, g, beta, z, snaps=None):
        """qkv [T, (2 k_heads + v_heads) * d] fp16 from the layer's convolution, g, beta [T, v_heads] fp32, z
        [T, v_heads, d]; `snaps` [T, v_heads, d, d] keeps the state after every token and leaves self.state alone."""
        T, kw = qkv.shape[0], self.kh * self.hd
        q, k, v = (x.unflatten(1, (-1, self.hd)) for x in (qkv[:, :kw], qkv[:, kw:2 * kw], qkv[:, 2 * kw:]))
        need = wz.gdn_delta_rule_workspace_bytes(T, self.kh, self.vh, self.hd)
        if need > self.ws.numel():
            self.ws = torch.empty(need, dtype=torch.uint8, device=qkv.device)
        o = torch.empty(T, self.vh, self.hd, dtype=F16, device=qkv.device)
        out = self.state if snaps is None else torch.empty_like(self.state)
        wz.gdn_delta_rule(q, k, v, g, beta, o, out, state_in=self.state, state_snaps=snaps, workspace=self.ws)
        y = torch.empty_like(o)
        wz.gdn_gated_norm(o, z, self.gamma, y, T, self.vh, self.hd)
        return y


def inputs(T, attn: AttentionMixer, gdn: GdnMixer, seed=0, device="cuda"):
    r = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=r, device=device)

    a = dict(q=randn(T, attn.qh, attn.hd).half(), k=randn(T, attn.kvh * attn.hd).half(), v=randn(T, attn.kvh * attn.hd).half())
    x = randn(T, (2 * gdn.kh + gdn.vh) * gdn.hd)
    b = dict(qkv=(x * torch.sigmoid(x)).half(), g=-0.05 * torch.exp(randn(T, gdn.vh)), beta=torch.sigmoid(randn(T, gdn.vh)),
             z=randn(T, gdn.vh, gdn.hd).half())
    return a, b


def run(prompt=4096, chunk=1024, decoded=8, device="cuda", **attn_kw):
    """Chunked prompt, decoded tokens, one verified tree; returns the outputs of both layers in order."""
    attn, gdn = AttentionMixer(device=device, **attn_kw), GdnMixer(device=device)
    a, b = inputs(prompt + decoded, attn, gdn, device=device)
    cuts = list(range(0, prompt, chunk)) + list(range(prompt, prompt + decoded + 1))
    ya, yb = [], []
    for lo, hi in zip(cuts, cuts[1:]):
        ya.append(attn.forward(*(a[n][lo:hi].clone() for n in ("q", "k", "v"))))
        yb.append(gdn.forward(*(b[n][lo:hi] for n in ("qkv", "g", "beta", "z"))))

    # a drafted tree of 4 nodes: 0 - 1 - 2 and 0 - 3; nodes 0, 1 are accepted
    n = 4
    mask = torch.tensor([[0b0001], [0b0011], [0b0111], [0b1001]], dtype=torch.int32, device=device)
    depth = torch.tensor([0, 1, 2, 1], dtype=torch.int32, device=device)
    q = torch.randn(n, attn.qh, attn.hd, device=device)
    k, v = (torch.randn(n, attn.kvh * attn.hd, device=device) for _ in range(2))
    tree = attn.verify(q, k, v, mask, depth)
    attn.accept(k[:2], v[:2])
    # the GDN layer sees the same drafts as a chain 0, 1, 2 and keeps the state after each: back to after node 1
    _, d = inputs(3, attn, gdn, seed=1, device=device)
    snaps = torch.empty(3, gdn.vh, gdn.hd, gdn.hd, device=device)
    gdn.forward(**d, snaps=snaps)
    gdn.state.copy_(snaps[1])
    return torch.cat(ya), torch.cat(yb), tree, attn, gdn


if __name__ == "__main__":
    ya, yb, tree, attn, gdn = run()
    torch.cuda.synchronize()
    print(f"attention {tuple(ya.shape)}, GDN {tuple(yb.shape)}, verified tree {tuple(tree.shape)}, "
          f"{int(attn.pos)} tokens committed, faults {wz.read_faults():#x}")
