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
