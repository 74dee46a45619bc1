"""A Qwen3 decoder over a cache of bounded size, in 64 bits: the plain decoder's layers, a portion of tokens after the other."""

from __future__ import annotations

import math

import torch

from . import kept_plain, qwen3_plain as plain


class Text:
    """One text under a policy: ``append`` runs a portion through all layers and returns its logits. ``gap``: the least relative distance seen
    between the weight of the last row that stayed and the first that went (how close a call an eviction was)."""

    def __init__(self, cfg, weights, policy):
        self.s = plain.settings(cfg)
        self.w = {k: v.double() for k, v in weights.items()}
        self.policy = policy
        K = self.s["kv_heads"]
        self.rows = [[dict(k=[], v=[], w=[], at=[]) for _ in range(K)] for _ in range(self.s["layers"])]
        self.seen = 0
        self.gap = math.inf

    def append(self, tokens):
        s, w = self.s, self.w
        ids = torch.as_tensor(list(tokens))
        T = len(ids)
        x = w["model.embed_tokens.weight"][ids]
        cos, sin = plain.rope_tables(s["head_dim"], self.seen + T, s["theta"])
        cos, sin = cos[self.seen:], sin[self.seen:]
        for i in range(s["layers"]):
            p = f"model.layers.{i}."
            x = x + self._attention(plain.rms_norm(x, w[p + "input_layernorm.weight"], s["eps"]), p + "self_attn.", i, cos, sin)
            x = x + plain.swiglu(plain.rms_norm(x, w[p + "post_attention_layernorm.weight"], s["eps"]), w, p + "mlp.")
        self.seen += T
        h = plain.rms_norm(x, w["model.norm.weight"], s["eps"])
        out = w["model.embed_tokens.weight"] if (s["tied"] or "lm_head.weight" not in w) else w["lm_head.weight"]
        return h @ out.T

    def _attention(self, h, prefix, layer, cos, sin):
        s, w, policy = self.s, self.w, self.policy
        T, H, K, hd = h.shape[0], s["heads"], s["kv_heads"], s["head_dim"]

        def lin(name):
            y = h @ w[prefix + name + ".weight"].T
            b = w.get(prefix + name + ".bias")
            return y if b is None else y + b

        q, k, v = (lin(n + "_proj").view(T, -1, hd).transpose(0, 1) for n in "qkv")
        if prefix + "q_norm.weight" in w:
            q, k = plain.rms_norm(q, w[prefix + "q_norm.weight"], s["eps"]), plain.rms_norm(k, w[prefix + "k_norm.weight"], s["eps"])
        q, k = plain.apply_rope(q, cos, sin), plain.apply_rope(k, cos, sin)
        y = torch.zeros((T, H, hd), dtype=torch.float64)
        G = H // K
        for kh in range(K):
            r = self.rows[layer][kh]
            past = len(r["k"])
            r["k"] += list(k[kh])
            r["v"] += list(v[kh])
            r["w"] += [0.0] * T
            r["at"] += [self.seen + i for i in range(T)]
            keys, values = torch.stack(r["k"]), torch.stack(r["v"])
            n = past + T
            gained = torch.zeros(n, dtype=torch.float64)
            for i in range(T):
                see = kept_plain.visible(past + i, n, policy.window, policy.first)
                for head in range(kh * G, kh * G + G):
                    a = torch.softmax(keys[see] @ q[head, i] / math.sqrt(hd), dim=0)
                    y[i, head] = a @ values[see]
                    gained[see] += a
            r["w"] = [x + float(g) for x, g in zip(r["w"], gained)]
            if policy.budget and n > policy.budget:
                seen = self.seen + T
                source, at = kept_plain.evict(r["w"], r["at"], n, n, seen, policy.budget, policy.first, policy.latest)
                free = [j for j in range(n) if policy.first <= r["at"][j] < seen - policy.latest]
                stays = [r["w"][j] for j in free if j in set(source)]
                goes = [r["w"][j] for j in free if j not in set(source)]
                if stays and goes:
                    self.gap = min(self.gap, (min(stays) - max(goes)) / max(max(goes), 1e-30))
                r["k"], r["v"], r["w"], r["at"] = ([r[name][j] for j in source] for name in ("k", "v", "w", "at"))
        return y.reshape(T, H * hd) @ w[prefix + "o_proj.weight"].T
