"""Speculative decoding on one model: the segment-tree Decoder drafts, the dense model verifies over the 8-bit paged cache.

The reference decodes token by token, sparse or dense (engine.py:149-177). Here the sparse engine's cheap steps propose a few
tokens, one dense pass over all of them (PagedDecoder: paged_append, paged_attn) gives the target's probabilities, and
verify_drafts keeps the drafts that stand and draws the next token, so that what comes out is distributed as the dense
model's own sampling."""
import torch

from . import _ops
from .paged import PagedKV, PagePool, _workspace_bytes, paged_append, paged_attn, paged_attn_workspace, verify_drafts


class PagedDecoder:
    """The dense model (the whole prefix in every layer) over an 8-bit paged cache, for any number of new tokens of each
    sequence at a time: a prompt, a chunk of one, a run of drafts, a single token.

    W: a decoder weight dict (engine.weights_from_ours / weights_from_nanogpt). max_len: positions of a sequence (at most the
    model's position table). n_pages: pages of the pool, shared by the layers' tables (default: enough for every sequence at
    max_len). rotation: (cos, sin) of paged.rotation_table for models that rotate their keys and queries.
    max_new: new tokens of a sequence in a call that the workspace is made for (it grows where a call has more)."""

    def __init__(self, W, n_layer, n_head, n_embd, batch=1, max_len=None, page=64, n_pages=None, dtype=torch.bfloat16,
                 dev='cuda', rotation=None, max_new=8):
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError('PagedDecoder: bfloat16 or float16 (got %s)' % dtype)
        self.dev, self.dtype, self.rotation = torch.device(dev), dtype, rotation
        cast = lambda t: t.to(device=self.dev, dtype=dtype).contiguous()
        norm = lambda t: t.to(self.dev, torch.float32).contiguous()
        self.W = dict(wte=cast(W['wte']), wpe=cast(W['wpe']), ln_f=norm(W['ln_f']),
                      layers=[dict(ln1=norm(L['ln1']), c_attn=cast(L['c_attn']), c_proj=cast(L['c_proj']), ln2=norm(L['ln2']),
                                   c_fc=cast(L['c_fc']), c_mlp=cast(L['c_mlp'])) for L in W['layers'][:n_layer]])
        self.H, self.C, self.dh, self.batch = n_head, n_embd, n_embd // n_head, batch
        self.max_len = int(max_len or W['wpe'].shape[0])
        if self.max_len > W['wpe'].shape[0]:
            raise ValueError('PagedDecoder: max_len %d above the position table\'s %d' % (self.max_len, W['wpe'].shape[0]))
        if rotation is not None and (rotation[0].shape[0] < self.max_len or 2 * rotation[0].shape[1] > self.dh):
            raise ValueError('PagedDecoder: a rotation of %d positions and %d dims for %d positions of %d' % (
                rotation[0].shape[0], 2 * rotation[0].shape[1], self.max_len, self.dh))
        per_seq = -(-self.max_len // page)
        self.pool = PagePool(n_pages or batch * per_seq, batch, per_seq, page, self.dev)
        self.caches = [PagedKV.empty(self.pool.n_pages, n_head, self.dh, self.pool.table, page, dtype) for _ in range(n_layer)]
        self.pos = [0] * batch     # positions that each sequence holds
        self._floor = [0] * batch  # and how far back it can be cut: the start of the page before the furthest one written
        self._start = {}
        self._ws = None
        self._grow(max_new)

    def _grow(self, n):
        """One workspace for the calls of every length (they run one after the other), as large as the largest one asked for."""
        sizes = self.batch, self.H, self.H, self.dh, n
        if self._ws is None or _workspace_bytes(*sizes) > self._ws.nbytes:
            self._ws = paged_attn_workspace(*sizes, self.dev)

    def _plan(self, n):
        """Row offsets of n rows a sequence (kept for the lengths that come up most, drafts and single tokens: a call less), and
        the attention's workspace."""
        if n not in self._start:
            if len(self._start) >= 16:
                self._start.clear()
            self._start[n] = torch.arange(self.batch + 1, device=self.dev, dtype=torch.int32) * n
            self._grow(n)
        return self._start[n], self._ws

    def reset(self):
        """Empties every sequence and gives its pages back."""
        for b in range(self.batch):
            self.pool.release(b)
        self.pos, self._floor = [0] * self.batch, [0] * self.batch

    @torch.no_grad()
    def forward(self, tok):
        """Feeds tok (batch, n) (whole numbers, on any device) at the sequences' next positions and returns the logits (batch, n,
        vocabulary) after each."""
        tok = tok.to(self.dev, torch.int64)
        B, n = tok.shape
        if B != self.batch:
            raise ValueError('PagedDecoder: %d sequences for a batch of %d' % (B, self.batch))
        if max(self.pos) + n > self.max_len:
            raise ValueError('PagedDecoder: position %d above max_len %d' % (max(self.pos) + n, self.max_len))
        self.pool.reserve([p + n for p in self.pos])
        start, ws = self._plan(n)
        pos = torch.tensor(self.pos, dtype=torch.int32).to(self.dev, non_blocking=True)
        at = (pos[:, None] + torch.arange(n, device=self.dev, dtype=torch.int32)).reshape(-1)
        W, C, H, dh, N = self.W, self.C, self.H, self.dh, B * n
        x = torch.empty(N, C, device=self.dev, dtype=torch.float32)
        h = torch.empty(N, C, device=self.dev, dtype=self.dtype)
        _ops.embed_ln(W['wte'], W['wpe'], tok.reshape(-1).contiguous(), at, W['layers'][0]['ln1'], x, h)
        for i, L in enumerate(W['layers']):
            qkv = h @ L['c_attn'].t()
            q, k, v = [qkv[:, j * C:(j + 1) * C].view(N, H, dh) for j in range(3)]
            q = paged_append(self.caches[i], k, v, start, pos, n, q=q, rotation=self.rotation)
            att = paged_attn(self.caches[i], q, start, pos, n, ws=ws)
            _ops.add_ln(x, att.view(N, C) @ L['c_proj'].t(), L['ln2'], h)
            f = _ops.gelu_(h @ L['c_fc'].t())
            _ops.add_ln(x, f @ L['c_mlp'].t(), W['layers'][i + 1]['ln1'] if i + 1 < len(W['layers']) else W['ln_f'], h)
        self.pos = [p + n for p in self.pos]
        page = self.pool.page
        self._floor = [max(f, ((p - 1) // page - 1) * page) for f, p in zip(self._floor, self.pos)]
        return (h @ W['wte'].t()).view(B, n, -1)

    def cut_back(self, pos):
        """Drops positions from pos[b] on (rejected drafts). A sequence can lose what is still in 16 bits: back to the start of
        the page before the furthest one written."""
        if len(pos) != self.batch:
            raise ValueError('PagedDecoder: %d lengths for a batch of %d' % (len(pos), self.batch))
        for b, (old, new) in enumerate(zip(self.pos, pos)):
            if not max(0, self._floor[b]) <= new <= old:
                raise ValueError('PagedDecoder: sequence %d cannot go from %d back to %d positions' % (b, old, new))
        self.pos = list(pos)


class SpeculativeDecoder:
    """draft: an engine.Decoder (mode 'seg') over the same vocabulary; target: a PagedDecoder, both of one batch size and both
    prefilled by prefill(). Each step drafts `n_draft` tokens of every sequence (fewer where the longest one nears the end of
    either cache, none for the last position) and verifies them. temperature 0 is greedy.
    generator: where the draws come from (a CUDA generator; default: torch's)."""

    def __init__(self, draft, target, n_draft=4, temperature=1.0, generator=None):
        if draft.batch != target.batch:
            raise ValueError('SpeculativeDecoder: draft batch %d, target batch %d' % (draft.batch, target.batch))
        if not 1 <= n_draft < target.pool.page:
            raise ValueError('SpeculativeDecoder: n_draft must be in [1, %d)' % target.pool.page)
        cfg = draft.cfg
        if cfg is not None and cfg.beam_mode == 'pred' and cfg.global_pool:
            raise ValueError('SpeculativeDecoder: a budget head over the running key mean cannot take drafts back')
        self.draft, self.target, self.G = draft, target, n_draft
        self.room = min(target.max_len, draft.cap, draft.W['wpe'].shape[0])  # positions that both hold
        self.temperature, self.generator = float(temperature), generator
        self.last = None     # (batch,) the newest token of each sequence, not fed yet
        self.accepted = 0    # drafts that stood so far, of all sequences
        self.drafted = 0

    def _probs(self, logits):
        if self.temperature == 0:
            return torch.nn.functional.one_hot(logits.argmax(-1), logits.shape[-1]).float()
        return torch.softmax(logits.float() / self.temperature, -1)

    @torch.no_grad()
    def prefill(self, idx):
        """Runs new prompts idx (batch, T) through both models, whatever they held before; returns the first new token of each
        sequence."""
        if idx.shape[1] > self.room:
            raise ValueError('SpeculativeDecoder: a prompt of %d positions for caches of %d' % (idx.shape[1], self.room))
        self.target.reset()
        self.draft.prefill(idx)
        logits = self.target.forward(idx.to(self.target.dev))[:, -1]
        self.last = torch.multinomial(self._probs(logits), 1, generator=self.generator)[:, 0]
        return self.last

    @torch.no_grad()
    def step(self):
        """One round: the new tokens of each sequence (a list of lists, 1 to n_draft + 1 of them). Raises ValueError, with nothing
        run, when a sequence has no position left."""
        B, dev = self.draft.batch, self.target.dev
        base = list(self.target.pos)
        left = self.room - max(base)  # the newest token takes one position, each draft another
        if left < 1:
            raise ValueError('SpeculativeDecoder: a sequence holds all %d positions' % self.room)
        G = min(self.G, left - 1)
        tok, drafts, probs = self.last, [], []
        at = torch.tensor(base, dtype=torch.int32).to(dev)
        for i in range(G + 1):  # the last round only puts the last draft into the draft's cache
            logits, _ = self.draft.step(tok, at + i)
            if i < G:
                q = self._probs(logits.view(B, -1))
                tok = torch.multinomial(q, 1, generator=self.generator)[:, 0]
                drafts.append(tok)
                probs.append(q)
        drafts = torch.stack(drafts, 1) if G else self.last.new_empty(B, 0)
        p = self._probs(self.target.forward(torch.cat([self.last[:, None], drafts], 1)))
        u = torch.rand(B, G + 1, device=dev, generator=self.generator)
        tokens, accepted = verify_drafts(p, torch.stack(probs, 1) if G else p[:, :0], drafts, u)
        self.last = tokens.gather(1, accepted[:, None].long())[:, 0]
        n = accepted.tolist()
        self.target.cut_back([b + 1 + a for b, a in zip(base, n)])
        self.accepted += sum(n)
        self.drafted += B * G
        return [t[:a + 1] for t, a in zip(tokens.tolist(), n)]
