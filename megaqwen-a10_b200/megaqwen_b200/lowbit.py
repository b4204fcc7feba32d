"""Batched greedy decode in low-bit integers: INT8 products (`Int8Linear`) and a 4-bit KV cache (`KV4Cache`).

`LowBitDecoder` runs the model with the operators a long-context server needs next to the fused decoders: it takes the
INT8 weights of an `A10Int8MegakernelDecoder`, quantises activations to 8 bits per token, and keeps K and V in 4 bits,
so that 64 sequences of 32,768 positions take 68 GB instead of the 240 GB of a bf16 cache.  Prompts go through in
chunks (all sequences of the batch at once, each with its own length); every step decodes one token for each sequence.

Norms, the rotation and SiLU are torch operations in fp32; the residual stream is bf16 as in the fused decoders.
"""
import torch

from . import _lib
from .config import HEAD_DIM, HIDDEN_SIZE, INTERMEDIATE_SIZE, KV_SIZE, NUM_KV_HEADS, NUM_Q_HEADS, Q_SIZE, RMS_EPS, VOCAB_SIZE
from .kv4 import KV4Cache
from .linear8 import Int8Linear


def _rms(x, weight):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + RMS_EPS) * weight.float()).to(torch.bfloat16)


def _rotate(x, cos, sin):
    """Split-half rotation of [B, T, heads, 128] with cos, sin [B, T, 1, 128]."""
    x = x.float()
    half = HEAD_DIM // 2
    return (x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin).to(torch.bfloat16)


class LowBitDecoder:
    def __init__(self, weights, batch, max_seq_len, group=32, page_size=64, page_table=None, num_pages=None):
        """weights: an A10Int8MegakernelDecoder; max_seq_len <= the rows of its RoPE tables.  group, page_size, page_table,
        num_pages: of the KV4Cache."""
        if not 1 <= max_seq_len <= weights.cos_table_.shape[0]:
            raise ValueError("max_seq_len out of range")
        self.w, self.device, self.max_seq_len = weights, weights.device, max_seq_len
        self.cache = KV4Cache(weights.num_layers_, batch, max_seq_len, NUM_KV_HEADS, HEAD_DIM, group, page_size, page_table,
                              num_pages, weights.device)
        flat, sc = weights.layer_weights_flat_, weights.layer_scales_
        self.layers = []
        for i in range(weights.num_layers_):
            t, s = flat[i * 11:i * 11 + 11], sc[i * 7:i * 7 + 7]   # the constructor's order
            stack = lambda ws, ss: Int8Linear(torch.cat(ws, 0), torch.cat(ss, 0))
            self.layers.append({"norm1": t[0], "qkv": stack(t[1:4], s[0:3]), "qn": t[4], "kn": t[5], "o": Int8Linear(t[6], s[3]),
                                "norm2": t[7], "gu": stack(t[8:10], s[4:6]), "down": Int8Linear(t[10], s[6])})
        self.lm = Int8Linear(weights.lm_head_weight_, weights.lm_head_scale_)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.tokens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self._host_lengths = [0] * batch
        self.status_ = torch.zeros(2, dtype=torch.int32, device=self.device)   # MQ_DEV_BAD_TOKEN and the sequence
        torch.cuda.current_stream(self.device).synchronize()

    def reset(self):
        self.lengths.zero_()
        self._host_lengths = [0] * self.cache.batch

    def _forward(self, ids, counts):
        """ids int [B, T], counts int32 [B] or None: appends the tokens and returns the residual stream [B, T, hidden]."""
        B, T = ids.shape
        start = self.lengths.clone()
        self.lengths += T if counts is None else counts
        pos = (start[:, None] + torch.arange(T, device=self.device)).clamp_(max=self.max_seq_len - 1)
        cos, sin = (t[pos].float()[:, :, None] for t in (self.w.cos_table_, self.w.sin_table_))
        h = self.w.embed_weight_[ids]
        for i, L in enumerate(self.layers):
            qkv = L["qkv"](_rms(h, L["norm1"]))
            q, k, v = qkv.split((Q_SIZE, KV_SIZE, KV_SIZE), -1)
            q = _rotate(_rms(q.view(B, T, NUM_Q_HEADS, HEAD_DIM), L["qn"]), cos, sin)
            k = _rotate(_rms(k.view(B, T, NUM_KV_HEADS, HEAD_DIM), L["kn"]), cos, sin)
            self.cache.append(i, k, v.view(B, T, NUM_KV_HEADS, HEAD_DIM), start, counts)
            a = self.cache.attend(i, q, self.lengths, counts)
            h = h + L["o"](a.view(B, T, Q_SIZE))
            g, u = L["gu"](_rms(h, L["norm2"]), out_dtype=torch.float32).split(INTERMEDIATE_SIZE, -1)
            h = h + L["down"](torch.nn.functional.silu(g) * u, out_dtype=torch.bfloat16)
        return h

    def _logits(self, h):
        """fp32 logits of rows [B, hidden]."""
        return self.lm(_rms(h, self.w.final_norm_weight_), out_dtype=torch.float32)

    def prefill(self, prompts, chunk=64):
        """prompts: one non-empty list of token ids for each sequence; appends them in chunks and returns fp32 logits
        [B, vocab] of every sequence's last token.  `tokens` holds the greedy choices for `step`."""
        B = self.cache.batch
        if len(prompts) != B or any(len(p) == 0 for p in prompts):
            raise ValueError(f"{B} non-empty prompts expected")
        if any(t < 0 or t >= VOCAB_SIZE for p in prompts for t in p):
            raise ValueError("token out of range")
        if chunk < 1:
            raise ValueError("chunk must be positive")
        if any(n + len(p) > self.max_seq_len for n, p in zip(self._host_lengths, prompts)):
            raise ValueError("prompt exceeds max_seq_len")
        last = torch.empty((B, HIDDEN_SIZE), dtype=torch.bfloat16, device=self.device)
        for c0 in range(0, max(len(p) for p in prompts), chunk):
            counts = [min(chunk, max(0, len(p) - c0)) for p in prompts]
            T = max(counts)
            ids = torch.tensor([p[c0:c0 + n] + [0] * (T - n) for p, n in zip(prompts, counts)], device=self.device)
            h = self._forward(ids, torch.tensor(counts, dtype=torch.int32, device=self.device))
            ends = [b for b, p in enumerate(prompts) if 0 < len(p) - c0 <= chunk]
            if ends:
                last[ends] = h[ends, [counts[b] - 1 for b in ends]]
        self._host_lengths = [n + len(p) for n, p in zip(self._host_lengths, prompts)]
        logits = self._logits(last)
        self.tokens = logits.argmax(-1).int()
        return logits

    def _ids(self, tokens):
        """int32 [B] on the device from a list or tensor of token ids.  What is on the host is checked here; a bad
        one on the device becomes token 0 there and is left in the status word, without a synchronisation."""
        t = torch.as_tensor(tokens)
        if t.shape != (self.cache.batch,):
            raise ValueError("one token for each sequence expected")
        bad = ~((t >= 0) & (t < VOCAB_SIZE))               # before the cast to 32 bits, which could wrap
        if t.device.type == "cpu":
            if bad.any():
                raise ValueError("token out of range")
            return t.int().to(self.device)
        if t.device != self.device:
            raise ValueError(f"tokens: on {t.device}, expected {self.device}")
        first = bad.int().argmax().int()
        self.status_.copy_(torch.where(bad.any(), torch.stack([torch.full_like(first, _lib.MQ_DEV_BAD_TOKEN), first]), self.status_))
        return t.masked_fill(bad, 0).int()

    def step(self, tokens=None):
        """Appends one token for each sequence (default: the last greedy choices) and returns fp32 logits [B, vocab];
        `tokens` holds the new greedy choices.  No host synchronisation.  A token outside the vocabulary raises; one in a
        tensor on the device is reported by `check_device`, and its sequence's logits mean nothing."""
        if max(self._host_lengths) >= self.max_seq_len:
            raise ValueError("KV cache full")
        ids = self.tokens if tokens is None else self._ids(tokens)
        logits = self._logits(self._forward(ids[:, None], None)[:, 0])
        self._host_lengths = [n + 1 for n in self._host_lengths]
        self.tokens = logits.argmax(-1).int()
        return logits

    def generate(self, prompts, max_new_tokens):
        """Greedy continuation: one list of max_new_tokens ids for each prompt."""
        self.reset()
        self.prefill(prompts)
        out = [self.tokens]
        for _ in range(max_new_tokens - 1):
            self.step()
            out.append(self.tokens)
        self.check_device()
        return torch.stack(out, 1)[:, :max(0, max_new_tokens)].tolist()

    def check_device(self):
        """Raises (and clears the status) if a call met a token, position or page that does not exist, or a wait ran out."""
        code, info = self.status_.tolist()
        if code:
            self.status_.zero_()
            raise _lib.MQError(f"low-bit decoder: device error {code} ({_lib.MQ_DEV_ERRORS.get(code, '?')}, sequence {info})")
        self.cache.check_device()
        for L in self.layers:
            for n in ("qkv", "o", "gu", "down"):
                L[n].check_device()
        self.lm.check_device()
