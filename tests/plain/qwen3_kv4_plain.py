"""The Qwen3 decoder with keys and values as a cache in 4 bits holds them, plainly."""
import math

import torch

from . import kv4_plain as K
from . import qwen3_plain as P


def held(x):
    """[tokens, kv_heads, d] -> the values that their codes stand for."""
    return K.decode(*K.encode(x.double())).to(x.dtype)


def forward(cfg, w, tokens, dtype=torch.float64, cached=None):
    """Logits [tokens, vocab].  cached: per layer the keys and values that stand in a cache (used in place of the ones computed here); the result is then
    the logits and, per layer, the keys and values computed here before they are stored."""
    made = []
    T, H, KV, D = len(tokens), cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
    positions, inv = torch.arange(T), P.rope_inv_freq(cfg["theta"], D)
    x = w["model.embed_tokens.weight"].to(dtype)[torch.as_tensor(list(tokens))]
    for layer in range(cfg["layers"]):
        p = f"model.layers.{layer}."
        xn = P.rms_norm(x, w[p + "input_layernorm.weight"], cfg["eps"])
        q, k, v = ((xn @ w[p + f"self_attn.{n}_proj.weight"].to(dtype).T).view(T, h, D) for n, h in (("q", H), ("k", KV), ("v", KV)))
        q = P.rope(P.rms_norm(q, w[p + "self_attn.q_norm.weight"], cfg["eps"]), positions, inv)
        k = P.rope(P.rms_norm(k, w[p + "self_attn.k_norm.weight"], cfg["eps"]), positions, inv)
        made.append((k, v))
        k, v = (held(k), held(v)) if cached is None else (c.to(dtype) for c in cached[layer])
        att = P.causal_attention(q, k, v, 1.0 / math.sqrt(D)).reshape(T, H * D)
        x = x + att @ w[p + "self_attn.o_proj.weight"].to(dtype).T
        x = x + P.swiglu(P.rms_norm(x, w[p + "post_attention_layernorm.weight"], cfg["eps"]), w, p)
    head = w["model.embed_tokens.weight"] if (cfg["tied"] or "lm_head.weight" not in w) else w["lm_head.weight"]
    logits = P.rms_norm(x, w["model.norm.weight"], cfg["eps"]) @ head.to(dtype).T
    return logits if cached is None else (logits, made)


def greedy(cfg, w, prompt, n):
    """Greedy tokens, and how far the best logit was before the second each time."""
    seq, lead = list(prompt), []
    for _ in range(n):
        row = forward(cfg, w, seq)[-1]
        top = row.topk(2).values
        lead.append(float(top[0] - top[1]))
        seq.append(P.argmax_first(row))
    return seq[len(prompt):], lead
