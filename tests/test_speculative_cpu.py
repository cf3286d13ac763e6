"""Host logic of the paged decoder and of speculative decoding, with the kernels' wrappers replaced."""
import pytest
import torch


@pytest.fixture
def host_model(monkeypatch):
    """PagedDecoder on the host: its kernels do nothing; `seen` collects what the embedding gets (tokens, positions)."""
    from treeattn_b200 import _ops, speculative
    from treeattn_b200.config import Config
    from treeattn_b200.engine import weights_from_ours
    from treeattn_b200.model import GPT
    seen = []

    def embed(wte, wpe, tok, pos, w, x, h):
        seen.append((tok, pos))
        x.zero_()
        h.zero_()

    class Cache:
        @staticmethod
        def empty(*a, **k):
            return None

    monkeypatch.setattr(_ops, 'embed_ln', embed)
    monkeypatch.setattr(_ops, 'add_ln', lambda x, y, w, h: h.zero_())
    monkeypatch.setattr(_ops, 'gelu_', lambda x: x)
    monkeypatch.setattr(speculative, 'PagedKV', Cache)
    monkeypatch.setattr(speculative, 'paged_append', lambda c, k, v, start, pos, n, q=None, rotation=None: q)
    monkeypatch.setattr(speculative, 'paged_attn', lambda c, q, *a, **k: q.contiguous())
    cfg = Config(attn='seg', vocab_size=64, seq_len=128, n_layer=1, n_head=2, n_embd=32, neighbors=False)
    W = weights_from_ours(GPT(cfg).state_dict(), cfg)

    def make(batch=2, **kw):
        return speculative.PagedDecoder(W, 1, 2, 32, batch=batch, dev='cpu', page=16, **kw)

    make.seen, make.W, make.cfg = seen, W, cfg
    return make


@pytest.mark.parametrize('dtype', [torch.int32, torch.int16, torch.int64])
def test_token_ids_reach_the_embedding_as_int64(host_model, dtype):
    """The embedding kernel reads 64-bit ids: ids of any whole type, from any strides, come to it as those."""
    dec = host_model()
    tok = torch.arange(12).view(6, 2).t().to(dtype)
    dec.forward(tok)
    got, pos = host_model.seen[-1]
    assert got.dtype is torch.int64 and got.is_contiguous() and got.tolist() == tok.reshape(-1).tolist()
    assert pos.tolist() == list(range(6)) * 2


class Draft:
    """A draft model that says which positions it was fed, and refuses those beyond its cache as the device would."""

    def __init__(self, batch, cap, vocab, table=None):
        self.batch, self.cap, self.vocab, self.cfg, self.fed = batch, cap, vocab, None, []
        self.W = dict(wpe=torch.zeros(table or cap, 8))

    def prefill(self, idx):
        self.fed.append(list(range(idx.shape[1])))

    def step(self, tok, at):
        assert int(at.max()) < min(self.cap, self.W['wpe'].shape[0]), 'fed a position beyond its cache'
        self.fed.append(at.tolist())
        return torch.zeros(self.batch, self.vocab), None


def _verified(p, q, drafts, u, n_draft=None):
    """Every draft stands, token 1 follows."""
    B, G = drafts.shape
    assert p.shape[:2] == (B, G + 1) and q.shape[:2] == (B, G) and u.shape == (B, G + 1)
    return torch.cat([drafts, torch.ones(B, 1, dtype=torch.int64)], 1), torch.full((B,), G, dtype=torch.int32)


@pytest.mark.parametrize('max_len,cap,table', [(64, 64, 64), (64, 40, 64), (40, 64, 64), (64, 64, 40)])
def test_rounds_end_at_the_last_position(host_model, monkeypatch, max_len, cap, table):
    """No model is fed a position beyond the smaller cache; the last rounds draft fewer, the last position is used, and then a
    round is refused before anything runs."""
    from treeattn_b200 import speculative
    monkeypatch.setattr(speculative, 'verify_drafts', _verified)
    room = min(max_len, cap, table)
    target, draft = host_model(max_len=max_len), Draft(2, cap, 64, table)
    dec = speculative.SpeculativeDecoder(draft, target, 4)
    dec.prefill(torch.zeros(2, 20, dtype=torch.int64))
    assert [len(x) for x in dec.step()] == [5, 5]
    while target.pos[0] < room:
        assert 1 <= len(dec.step()[0]) <= 5
    assert target.pos == [room, room] and draft.fed[-1] == [room - 1, room - 1]
    fed, seen = len(draft.fed), len(host_model.seen)
    with pytest.raises(ValueError, match='all %d positions' % room):
        dec.step()
    assert (len(draft.fed), len(host_model.seen), target.pos) == (fed, seen, [room, room])
    with pytest.raises(ValueError, match='prompt of'):
        dec.prefill(torch.zeros(2, room + 1, dtype=torch.int64))
    assert len(draft.fed) == fed


def test_the_longest_sequence_sets_the_round(host_model, monkeypatch):
    """Uneven lengths: a round is as long as the longest sequence leaves room for."""
    from treeattn_b200 import speculative
    monkeypatch.setattr(speculative, 'verify_drafts', _verified)
    target, draft = host_model(max_len=32), Draft(2, 32, 64)
    dec = speculative.SpeculativeDecoder(draft, target, 4)
    dec.prefill(torch.zeros(2, 30, dtype=torch.int64))
    target.cut_back([30, 22])
    assert [len(x) for x in dec.step()] == [2, 2]
    assert target.pos == [32, 24]
    with pytest.raises(ValueError, match='all 32'):
        dec.step()


def test_a_second_prompt_starts_anew(host_model, monkeypatch):
    """prefill() begins both models at position 0 again, with every page of the last prompt free."""
    from treeattn_b200 import speculative
    monkeypatch.setattr(speculative, 'verify_drafts', _verified)
    target, draft = host_model(max_len=96, n_pages=12), Draft(2, 96, 64)
    dec = speculative.SpeculativeDecoder(draft, target, 4)
    for T in (85, 20, 90):
        dec.prefill(torch.zeros(2, T, dtype=torch.int64))
        assert target.pos == [T, T] and host_model.seen[-1][1].tolist() == list(range(T)) * 2
        dec.step()
        assert draft.fed[-5:] == [[T + i] * 2 for i in range(5)] and target.pos == [T + 5, T + 5]
        assert sorted(target.pool.free + sum(target.pool.owned, [])) == list(range(12))


def test_cut_back_wants_a_length_for_every_sequence(host_model):
    """Fewer lengths than sequences would leave the embedding fewer positions than rows."""
    dec = host_model(batch=3)
    dec.forward(torch.zeros(3, 9, dtype=torch.int64))
    for bad in ([8], [8, 8], [8] * 4):
        with pytest.raises(ValueError, match='lengths for a batch of 3'):
            dec.cut_back(bad)
    assert dec.pos == [9, 9, 9]
    dec.cut_back([8, 9, 0])
    dec.forward(torch.zeros(3, 2, dtype=torch.int64))
    assert host_model.seen[-1][1].tolist() == [8, 9, 9, 10, 0, 1]


def test_prompts_of_many_lengths_keep_one_workspace(host_model, monkeypatch):
    """What the decoder holds for its calls does not grow with the lengths it has seen: one workspace of the largest size, few row
    offsets, each call's workspace large enough for it."""
    from treeattn_b200 import speculative
    from treeattn_b200.paged import paged_attn_workspace
    given = []

    def attn(c, q, start, pos, n, ws=None, **k):
        assert start.tolist() == [0, n, 2 * n]
        given.append((n, ws))
        return q.contiguous()

    monkeypatch.setattr(speculative, 'paged_attn', attn)
    dec = host_model()
    lengths = [1, 5] + list(range(7, 120, 4)) + [1, 5, 100]
    for n in lengths:
        dec.reset()
        dec.forward(torch.zeros(2, n, dtype=torch.int64))
    need = {n: paged_attn_workspace(2, 2, 2, 16, n, 'cpu').nbytes for n in lengths}
    assert all(ws.nbytes >= need[n] for n, ws in given) and dec._ws.nbytes == max(need.values())
    held = [x for v in vars(dec).values() for x in (v.values() if isinstance(v, dict) else [v]) if torch.is_tensor(x)
            and x.dtype is torch.uint8]
    assert sum(x.nbytes for x in held) == max(need.values()) and len(dec._start) <= 16


def test_rotation_table_covers_the_context(host_model):
    """Positions beyond the tables would be left out of the cache; a rotation of more dims than a head has is refused at once too."""
    from treeattn_b200.paged import rotation_table
    host_model(max_len=100, rotation=rotation_table(100, 16, device='cpu'))
    for n, rot in ((99, 16), (128, 18)):
        with pytest.raises(ValueError, match='rotation of %d positions and %d dims' % (n, rot)):
            host_model(max_len=100, rotation=rotation_table(n, rot, device='cpu'))


def test_a_released_slot_has_no_adapter(host_model):
    """The next request in a slot that was released does not run with the last one's adapter; reset keeps the adapters, as documented."""
    from treeattn_b200.adapters import AdapterSet
    dec = host_model(batch=3, adapters=AdapterSet(2, 1, 32, rank=8, device='cpu'))
    for b, a in enumerate((1, 0, 1)):
        dec.set_adapter(b, a)
    dec.release(1)
    assert dec.which.tolist() == [1, -1, 1] and dec.pos == [0, 0, 0]
    dec.reset()
    assert dec.which.tolist() == [1, -1, 1]
    plain = host_model()
    plain.release(0)
    assert plain.which.tolist() == [-1, -1]


def test_a_refused_fork_changes_nothing(host_model, monkeypatch):
    """Neither lists that the pool refuses nor moves that the copy refuses (a cycle above its limit) leave a sequence half forked."""
    from treeattn_b200 import speculative
    from treeattn_b200._lib import TreeAttnError
    dec, copied = host_model(batch=3), []
    monkeypatch.setattr(speculative, 'paged_fork', lambda caches, src, dst: copied.append((src, dst)))
    dec.forward(torch.zeros(3, 40, dtype=torch.int64))
    state = lambda: ([list(o) for o in dec.pool.owned], list(dec.pool.free), list(dec.pool.refs), dec.pool.extra, dec.pool.table.tolist(),
                     list(dec.pos), list(dec._floor), dec.which.tolist())
    before = state()
    for src, dst in (([0], [3]), ([-1], [1]), ([0, 0], [1, 1]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            dec.fork(src, dst)
        assert state() == before and not copied

    def refuse(caches, src, dst):
        raise TreeAttnError('ta_record_copy: a cycle of 2048 moves (at most 2047)')

    monkeypatch.setattr(speculative, 'paged_fork', refuse)
    with pytest.raises(TreeAttnError):
        dec.fork([0, 1], [1, 0])
    assert state() == before
    monkeypatch.setattr(speculative, 'paged_fork', lambda caches, src, dst: copied.append((src, dst)))
    dec.fork([0, 1], [1, 2])
    # 1 shares the two full pages of 0; what 1 held has gone to 2 alone
    assert copied == [([0, 1], [1, 2])] and dec.pool.extra == 2
