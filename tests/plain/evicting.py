"""The plain Qwen3 decoder over a cache whose rows are evicted by the attention they have gathered: every layer and kv head on its
own, one sequence. numpy only, from the definition; no code is shared with the package."""
from __future__ import annotations

import numpy as np

from .model import PlainQwen3, linear, rms_norm, rope_apply, rope_table, swiglu
from .rows import kept_rows


class PlainEvicting(PlainQwen3):
    def start(self, limit, keep, recent, first):
        self.bound = (limit, keep, recent, first)
        self.pos = 0
        self.held = [[dict(k=np.zeros((0, self.HD)), v=np.zeros((0, self.HD)), m=np.zeros((0,))) for _ in range(self.KV)] for _ in range(self.L)]

    def step(self, tokens) -> np.ndarray:
        """Logits behind every one of the tokens; rows beyond the bound are evicted afterwards."""
        n, group = len(tokens), self.H // self.KV
        x = self.t["model.embed_tokens.weight"][np.asarray(tokens)].astype(np.float32)
        cos, sin = rope_table(self.HD, np.arange(self.pos, self.pos + n), self.theta)
        for i in range(self.L):
            t, p = self.t, f"model.layers.{i}."
            h = rms_norm(x, t[p + "input_layernorm.weight"], self.eps)
            q = linear(h, t[p + "self_attn.q_proj.weight"]).reshape(n, self.H, self.HD)
            k = linear(h, t[p + "self_attn.k_proj.weight"]).reshape(n, self.KV, self.HD)
            v = linear(h, t[p + "self_attn.v_proj.weight"]).reshape(n, self.KV, self.HD)
            q = rope_apply(rms_norm(q, t[p + "self_attn.q_norm.weight"], self.eps), cos, sin)
            k = rope_apply(rms_norm(k, t[p + "self_attn.k_norm.weight"], self.eps), cos, sin)
            a = np.zeros((n, self.H, self.HD), dtype=np.float64)
            for g in range(self.KV):
                c = self.held[i][g]
                past = len(c["m"])
                c["k"] = np.concatenate([c["k"], k[:, g]])
                c["v"] = np.concatenate([c["v"], v[:, g]])
                c["m"] = np.concatenate([c["m"], np.zeros((n,))])
                for h in range(g * group, (g + 1) * group):
                    s = q[:, h].astype(np.float64) @ c["k"].T.astype(np.float64) / np.sqrt(self.HD)
                    s = np.where(np.arange(past + n)[None, :] <= past + np.arange(n)[:, None], s, -np.inf)
                    w = np.exp(s - s.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    a[:, h] = w @ c["v"]
                    c["m"] += w.sum(0)
            x = x + linear(a.reshape(n, -1).astype(np.float32), t[p + "self_attn.o_proj.weight"])
            h = rms_norm(x, t[p + "post_attention_layernorm.weight"], self.eps)
            x = (x + linear(swiglu(linear(h, t[p + "mlp.gate_proj.weight"]), linear(h, t[p + "mlp.up_proj.weight"])),
                            t[p + "mlp.down_proj.weight"])).astype(np.float32)
        self.pos += n
        limit, keep, recent, first = self.bound
        for layer in self.held:
            for c in layer:
                if len(c["m"]) > limit:
                    r = kept_rows(c["m"].tolist(), len(c["m"]), keep, recent, first)
                    for name in c:
                        c[name] = c[name][r]
        head = self.t["model.embed_tokens.weight"] if self.tied else self.t["lm_head.weight"]
        return linear(rms_norm(x, self.t["model.norm.weight"], self.eps), head)
