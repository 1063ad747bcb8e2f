"""The text decoder over sessions that grow.

The aligner prefills a clip's whole sequence once (src/cpu_decoder.rs:283-547).
A live transcript or a corrected word only adds a few tokens to a sequence whose
prefix is already known, and such a step is bound by what it reads: the weights
and the cache.  Here the same decoder (the checkpoint's tensors, the geometry of
`synth.ModelConfig`) runs with its projections in 4 bits and its K/V cache in 8
bits, paged, and one step takes any number of new tokens, none included, for any
set of sessions:

    dec = SessionDecoder(cfg, weights, pages=4096)
    a, b = dec.open(), dec.open()
    hidden = dec.step({a: prompt_ids, b: other_ids})   # rows in that order
    hidden = dec.step({a: [next_id]})
    dec.close(b)

A layer is `w4_linear` (q, k and v as one), `kv_append` (q/k RMSNorm, rotation,
cache), `cache_attention`, `w4_linear` (output), and `w4_linear` twice for the
gated MLP; the norms and the gate between them are plain tensor operations.  How
many tokens a step takes, and the most of one session, bear on the order of sums:
a session beside others agrees with itself alone within rounding.
"""
from __future__ import annotations

from . import _lib
from . import rope

PAGE = 64


def quantise4(w, group: int = 128, dtype=None):
    """4-bit codes of w [N, K] as `w4_linear` takes them: (wq uint8 [N, K / 2],
    scales [N, K / group] of `dtype`, zeros uint8).  Each group's range, widened
    to hold 0, is cut in 15 steps; a weight is off by half a step at most, plus
    half a step at the range's end, where the zero point was rounded, plus what
    rounding the step to `dtype` takes from the range.  float16's steps below 2^-14
    are whole units of 2^-24, rounded up, so that groups of tiny weights keep them."""
    import torch
    dtype = dtype or torch.bfloat16
    N, K = w.shape
    if group not in (32, 64, 128) or K % group:
        raise ValueError("K a multiple of a group of 32, 64 or 128")
    g = w.float().reshape(N, K // group, group)
    lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    step, tiny = (hi - lo) / 15, torch.finfo(dtype).tiny
    if dtype is torch.float16:
        step, tiny = torch.where(step < tiny, (step * 2 ** 24).ceil() * 2 ** -24, step), 2 ** -24
    scales = step.clamp(min=tiny).to(dtype)
    s = scales.float()
    zeros = (-lo / s).round().clamp(0, 15)
    codes = ((g / s[..., None]).round() + zeros[..., None]).clamp(0, 15).to(torch.uint8).reshape(N, K)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales, zeros.to(torch.uint8)


class PageTable:
    """Which pages of the pools hold which session's tokens (host side)."""

    def __init__(self, pages: int):
        self._free = list(range(pages - 1, -1, -1))
        self._pages: dict = {}
        self._len: dict = {}
        self._next = 0

    def open(self) -> int:
        sid, self._next = self._next, self._next + 1
        self._pages[sid], self._len[sid] = [], 0
        return sid

    def close(self, sid: int) -> None:
        self._free += reversed(self._pages.pop(sid))
        del self._len[sid]

    def length(self, sid: int) -> int:
        return self._len[sid]

    def pages(self, sid: int) -> list:
        return self._pages[sid]

    def extend(self, news: dict) -> None:
        """Room for news[sid] more tokens of each session: all of it or, with a
        MemoryError, none."""
        want = {s: -(-(self._len[s] + n) // PAGE) - len(self._pages[s]) for s, n in news.items()}
        if sum(want.values()) > len(self._free):
            raise MemoryError(f"{sum(want.values())} pages of {PAGE} tokens wanted, {len(self._free)} free")
        for s, n in news.items():
            self._pages[s] += [self._free.pop() for _ in range(want[s])]
            self._len[s] += n

    def shrink(self, news: dict) -> None:
        """Takes back the last `extend`, which was of these."""
        for s, n in reversed(news.items()):
            self._len[s] -= n
            keep = -(-self._len[s] // PAGE)
            self._free += reversed(self._pages[s][keep:])
            del self._pages[s][keep:]


class _Linear:
    def __init__(self, w, group, dtype, device):
        self.wq, self.scales, self.zeros = (t.contiguous() for t in quantise4(w.to(device), group, dtype))

    def __call__(self, x):
        out = x.new_empty(x.shape[0], self.wq.shape[0])
        _lib.w4_linear(x, self.wq, self.scales, out, zeros=self.zeros)
        return out


def _norm(x, gain, eps, dtype):
    import torch
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * gain).to(dtype)


class SessionDecoder:
    """Decoder weights in 4 bits and the paged 8-bit cache of every layer.

    `weights` maps checkpoint names to bf16 bits (`synth.random_weights`,
    `synth.load_safetensors`) or tensors.  `pages` pages of 64 tokens are shared
    by all sessions.  Work is queued on the current stream.
    """

    def __init__(self, cfg, weights, *, pages: int, dtype=None, group: int = 128, device="cuda"):
        import torch
        self.cfg, self.dtype = cfg, dtype or torch.bfloat16
        self.device = torch.device(device)
        if cfg.head_dim not in (64, 128) or cfg.num_heads % cfg.num_kv_heads:
            raise ValueError("heads of 64 or 128, query heads a multiple of the K/V heads")

        def get(name):
            w = weights["model.language_model." + name] if name != "score.weight" else weights[name]
            if not torch.is_tensor(w):
                w = torch.from_numpy(w.view("int16").copy()).view(torch.bfloat16)
            return w.to(self.device)

        def linear(*names):
            return _Linear(torch.cat([get(n) for n in names]), group, self.dtype, self.device)

        self.embed = get("embed_tokens.weight").to(self.dtype)
        self.norm = get("norm.weight").float()
        self.head = linear("score.weight")
        self.layers = []
        shape = (pages, cfg.num_kv_heads, PAGE, cfg.head_dim)
        for i in range(cfg.num_layers):
            p = f"layers.{i}."
            a = p + "self_attn."
            self.layers.append(dict(
                norm1=get(p + "input_layernorm.weight").float(),
                norm2=get(p + "post_attention_layernorm.weight").float(),
                qn=get(a + "q_norm.weight").float(), kn=get(a + "k_norm.weight").float(),
                qkv=linear(a + "q_proj.weight", a + "k_proj.weight", a + "v_proj.weight"),
                o=linear(a + "o_proj.weight"),
                gate_up=linear(p + "mlp.gate_proj.weight", p + "mlp.up_proj.weight"),
                down=linear(p + "mlp.down_proj.weight"),
                kpool=torch.zeros(shape, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn),
                vpool=torch.zeros(shape, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn),
                kscale=torch.ones(shape[:2], device=self.device),
                vscale=torch.ones(shape[:2], device=self.device)))
        half = cfg.head_dim // 2
        cos, sin = rope.rope_tables(cfg.max_seq, cfg.head_dim, cfg.rope_theta)
        self.cos = torch.from_numpy(cos[:, :half].copy()).to(self.device)
        self.sin = torch.from_numpy(sin[:, :half].copy()).to(self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.table = PageTable(pages)

    def open(self) -> int:
        return self.table.open()

    def close(self, sid: int) -> None:
        self.table.close(sid)

    def _check(self, news: dict) -> None:
        for s, ids in news.items():
            if len(ids) and not 0 <= min(ids) <= max(ids) < self.cfg.vocab_size:
                raise ValueError("a token id outside the vocabulary")
            if self.table.length(s) + len(ids) > self.cfg.max_seq:
                raise ValueError("a session longer than max_seq")

    def _maps(self, news: dict):
        """The step's token ids and sequence maps, in one copy to the device."""
        import torch
        sids = list(news)
        ids = [t for s in sids for t in news[s]]
        pages = [self.table.pages(s) for s in sids]
        wide = max([len(p) for p in pages] + [1])
        starts, lens = [0], [self.table.length(s) for s in sids]
        for s in sids:
            starts.append(starts[-1] + len(news[s]))
        flat = ids + starts + lens + [x for p in pages for x in p + [0] * (wide - len(p))]
        host = torch.tensor(flat, dtype=torch.int32)
        if self.device.type == "cuda":
            host = host.pin_memory()
        d = host.to(self.device, non_blocking=True)
        cut = [len(ids), len(starts), len(lens)]
        ids, q_start, kv_len, tab = d.split(cut + [len(flat) - sum(cut)])
        maps = dict(q_start=q_start, kv_len=kv_len, block_tab=tab.view(len(sids), wide))
        return ids, maps, max(len(v) for v in news.values()), max(lens)

    def step(self, news: dict):
        """Final hidden states (after the last norm) of the new tokens, in the
        order of `news`, a map from session to its new token ids.  A step that
        raises leaves the sessions with the tokens that they had."""
        import torch
        if not news:
            return torch.empty(0, self.cfg.hidden_size, dtype=self.dtype, device=self.device)
        self._check(news)
        sizes = {s: len(ids) for s, ids in news.items()}
        self.table.extend(sizes)
        try:
            return self._run(news)
        except BaseException:
            # What is queued still writes to the new slots, ahead of whatever is
            # queued next; slots past a session's length are never read.  A page
            # that was begun may keep the larger scale that a new value asked for.
            self.table.shrink(sizes)
            raise

    def _run(self, news: dict):
        import torch
        cfg = self.cfg
        ids, maps, max_q, max_kv = self._maps(news)
        nq, nkv, hd, eps = cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, cfg.rms_norm_eps
        x = self.embed[ids.long()].float()  # the residual stream stays in 32 bits
        seq = (maps["q_start"], maps["kv_len"], maps["block_tab"])
        for L in self.layers:
            qkv = L["qkv"](_norm(x, L["norm1"], eps, self.dtype))
            q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
            pool = (L["kpool"], L["vpool"])
            _lib.kv_append(q, k, v, q, *seq, *pool, kscale=L["kscale"], vscale=L["vscale"], cos=self.cos,
                           sin=self.sin, qn=L["qn"], kn=L["kn"], eps=eps, max_q=max_q,
                           status=self.status, validate=False)
            out = q.new_empty(q.shape)
            _lib.cache_attention(q, *seq, *pool, L["kscale"], L["vscale"], out, max_q=max_q,
                                 max_kv=max_kv, status=self.status, validate=False)
            x = x + L["o"](out).float()
            gate, up = L["gate_up"](_norm(x, L["norm2"], eps, self.dtype)).float().chunk(2, 1)
            x = x + L["down"]((torch.nn.functional.silu(gate) * up).to(self.dtype)).float()
        return _norm(x, self.norm, eps, self.dtype)

    def labels(self, hidden):
        """Scores of the timestamp head, [T, num_labels]."""
        return self.head(hidden)

    def check(self) -> None:
        """Waits for the queued work; QaError if a kernel refused a map."""
        if int(self.status):
            raise _lib.QaError(_lib.QA_ERR_ARG, "a sequence map was refused on the device")
