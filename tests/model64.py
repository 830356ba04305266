"""The Gemma 3 decode step in 64 bits over a cache as kv8_ref.py defines it (or an exact one), written from the published
operations (src/gemma3.cpp:1462-1882 for their order): one sequence, one token at a time."""
import numpy as np

import gguf
import kv8_ref


class Model64:
    def __init__(self, path, kv8=True):
        f = gguf.GgufFile.open(path)
        g = lambda k: f.meta_u64("gemma3." + k)  # noqa: E731
        self.d, self.n_layers, self.H = g("embedding_length"), g("block_count"), g("attention.head_count")
        self.hd, self.window = g("attention.key_length"), g("attention.sliding_window") or 0
        self.eps = f.meta_f64("gemma3.attention.layer_norm_rms_epsilon")
        self.base = [1.0e4, f.meta_f64("gemma3.rope.freq_base") or 1.0e6]

        def q8(name):
            t = f.tensors[name]
            b = np.frombuffer(f.tensor_bytes(name), np.uint8).reshape(-1, 34)
            s = b[:, :2].copy().view(np.float16).astype(np.float64)
            return (s * b[:, 2:].copy().view(np.int8)).reshape(t.dims[1], t.dims[0])

        f32 = lambda n: np.asarray(f.read_f32(n), np.float64)  # noqa: E731
        self.emb, self.out_norm = q8("token_embd.weight"), f32("output_norm.weight")
        mats = ("attn_q", "attn_k", "attn_v", "attn_output", "ffn_gate", "ffn_up", "ffn_down")
        norms = ("attn_norm", "attn_q_norm", "attn_k_norm", "post_attention_norm", "ffn_norm", "post_ffw_norm")
        self.blocks = [({m: q8(f"blk.{l}.{m}.weight") for m in mats}, {n: f32(f"blk.{l}.{n}.weight") for n in norms})
                       for l in range(self.n_layers)]
        self.kv8 = kv8
        self.reset()

    def reset(self):
        self.pos = 0
        # per block: the entries' keys and values as they entered (fp32), and the weights they got so far
        self.kv = [[np.zeros((0, 1, self.hd), np.float32)] * 2 for _ in self.blocks]
        self.w = [np.zeros(0) for _ in self.blocks]

    def whole(self, l):
        return (l + 1) % 6 == 0 or not self.window

    def _rms(self, x, w):
        return x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + self.eps) * w

    def _rope(self, x, whole):
        half = self.hd // 2
        a = self.pos * self.base[whole] ** (-2.0 * np.arange(half) / self.hd)
        c, s = np.cos(a), np.sin(a)
        x0, x1 = x[..., :half], x[..., half:]
        return np.concatenate([x0 * c - x1 * s, x1 * c + x0 * s], axis=-1)

    def step(self, token):
        """Logits of the next position; also weighs the entries of the blocks that attend to all."""
        h = self.emb[token] * np.float64(np.sqrt(np.float32(self.d)))
        for l, (W, N) in enumerate(self.blocks):
            x = self._rms(h, N["attn_norm"])
            glob = (l + 1) % 6 == 0
            q = self._rope(self._rms((W["attn_q"] @ x).reshape(self.H, self.hd), N["attn_q_norm"]), glob)
            k = self._rope(self._rms((W["attn_k"] @ x).reshape(1, self.hd), N["attn_k_norm"]), glob)
            v = (W["attn_v"] @ x).reshape(1, self.hd)
            ks, vs = (np.concatenate([a, b.astype(np.float32)[None]]) for a, b in zip(self.kv[l], (k, v)))
            self.kv[l] = [ks, vs]
            see = (lambda a: kv8_ref.stored(a)) if self.kv8 else (lambda a: a.astype(np.float64))
            o, w, _ = kv8_ref.attend(q[None], see(ks), see(vs), len(ks) - 1, float(np.float32(1.0 / np.sqrt(np.float32(self.hd)))),
                                     window=0 if self.whole(l) else self.window)
            self.w[l] = np.concatenate([self.w[l], [0.0]]) + w[0]
            h = h + self._rms(W["attn_output"] @ o.reshape(-1), N["post_attention_norm"])
            x = self._rms(h, N["ffn_norm"])
            g = W["ffn_gate"] @ x
            g = 0.5 * g * (1.0 + np.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3))) * (W["ffn_up"] @ x)
            h = h + self._rms(W["ffn_down"] @ g, N["post_ffw_norm"])
        self.pos += 1
        return self.emb @ self._rms(h, self.out_norm)

    def evict(self, keep, recent):
        for l in range(self.n_layers):
            if self.whole(l):
                at = kv8_ref.keep_rule(self.w[l], keep, recent)
                self.kv[l] = [kv8_ref.stored(a)[at] for a in self.kv[l]]
                self.w[l] = self.w[l][at]
