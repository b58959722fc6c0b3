"""Models over a 4-bit KV cache (tmg_cache_new_kv4, tmg_generate_kv4): the
cached rows against a float64 textbook decoder's, quantized from their
definition (kv4ref.py), and the logits against the same decoder reading the
cached rows, so that a key on the border between two codes is not held against
the logits behind it."""
import ctypes as C
import dataclasses

import numpy as np
import pytest

import kv4ref as R
from conftest import model_root
from textbook import TextbookLlama

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import tinyminigo_amd as T
    return T


class Decoder(TextbookLlama):
    """Logits and, per layer, f64 keys and values of `tokens`, with attention
    over the given keys and values kv[layer] = (k, v) [tokens][nkv][hd]."""

    def over(self, tokens, kv):
        n = len(tokens)
        pos = np.arange(n, dtype=np.float64)
        x, own = self.embed[np.asarray(tokens)], []
        for L, (kc, vc) in zip(self.layers, kv):
            h = self.rmsnorm(x, L["n1"])
            q = self.rope((h @ L["q"].T).reshape(n, self.nq, self.hd), pos)
            own.append((self.rope((h @ L["k"].T).reshape(n, self.nkv, self.hd), pos),
                        (h @ L["v"].T).reshape(n, self.nkv, self.hd)))
            out = np.empty((n, self.nq, self.hd))
            late = np.triu(np.full((n, n), -np.inf), k=1)
            for hh in range(self.nq):
                g = hh // (self.nq // self.nkv)
                s = q[:, hh] @ kc[:, g].T / np.sqrt(self.hd) + late
                s = np.exp(s - s.max(-1, keepdims=True))
                out[:, hh] = s / s.sum(-1, keepdims=True) @ vc[:, g]
            x = x + out.reshape(n, -1) @ L["o"].T
            h = self.rmsnorm(x, L["n2"])
            g, u = h @ L["g"].T, h @ L["u"].T
            x = x + (g / (1.0 + np.exp(-g)) * u) @ L["d"].T
        return self.rmsnorm(x, self.norm) @ self.lm.T, own


SHAPES = {  # hidden, layers, query heads, KV heads, head dim, intermediate
    "hd16": (64, 2, 4, 2, 16, 128),
    "hd32": (128, 2, 8, 1, 32, 256),
    "hd64": (256, 2, 4, 4, 64, 320),
    "hd128": (256, 2, 4, 2, 128, 512),
    "hd256": (256, 1, 4, 1, 256, 512),
}


@pytest.fixture(scope="module", params=list(SHAPES))
def model(request, T):
    from oracle import oracle as O
    from tinyminigo_amd import workloads as W
    H, L, nq, nkv, hd, inter = SHAPES[request.param]
    w = dataclasses.replace(W.TINY, name=f"tiny-kv4-{request.param}", hidden_size=H, num_hidden_layers=L,
                            num_attention_heads=nq, num_key_value_heads=nkv, head_dim=hd, intermediate_size=inter,
                            weight_seed=31)
    path = W.ensure_model(w, model_root())
    m = T.Model.load(path)
    return m, Decoder(m.config, O.load_safetensors(path)), w


def check(m, tb, cache, tokens, logits):
    """logits {position: row} of a session over `tokens` in `cache`.  The
    projections leave a key or value up to some 2e-6 of its size from f64's, so
    only one within that of a border may have the next code: less than 1 in
    200."""
    n, c = len(tokens), m.config
    kv = [tuple(x.reshape(n, c.num_key_value_heads, c.head_dim).astype(np.float64)
                for x in (cache.keys_flat(l), cache.values_flat(l))) for l in range(c.num_hidden_layers)]
    ref, own = tb.over(tokens, kv)
    for l in range(c.num_hidden_layers):
        for got, x in zip(kv[l], own[l]):
            code, byte = R.quantize(x.astype(np.float32))
            off = got != R.values(code, byte)
            assert off.mean() < 0.005, f"layer {l}: {off.mean():.4f} of the values differ"
            # by a code's spacing at most (2 s, the largest)
            s = np.exp2(byte.astype(np.float64) - 127).repeat(c.head_dim // byte.shape[-1], -1)
            assert (np.abs(got - R.values(code, byte)) <= 2 * s).all()
    for p, row in logits.items():
        d = np.abs(row - ref[p])
        assert (d <= 2e-3 + 1e-3 * np.abs(ref[p])).all(), f"position {p}: {d.max():.3g}"


@pytest.mark.parametrize("turns", [(1,), (16,), (5, 1, 40), (70, 30, 2)])
def test_session(T, model, turns):
    """Turns of forward_seq with decode steps between them."""
    m, tb, w = model
    cache = m.new_cache(sum(turns) + 4 * len(turns) + 3, kv4=True)
    tokens, logits = [], {}
    for i, n in enumerate(turns):
        ids = [int(t) for t in T.synth_tokens(90 + i, n, w.vocab_size)]
        row = m.forward_seq(ids, cache)
        tokens += ids
        logits[len(tokens) - 1] = row
        for _ in range(4):
            t = int(np.argmax(row))
            row = m.forward_token(t, cache)
            tokens.append(t)
            logits[len(tokens) - 1] = row
    assert cache.total_len() == len(tokens)
    check(m, tb, cache, tokens, logits)


def test_generate_is_the_session(T, model):
    m, tb, w = model
    prompt = [int(t) for t in T.synth_tokens(7, 33, w.vocab_size)]
    cache = m.new_cache(80, kv4=True)
    row, want = m.forward_seq(prompt, cache), []
    for _ in range(20):
        want.append(int(np.argmax(row)))
        row = m.forward_token(want[-1], cache)
    got = T.generate(m, prompt, T.GenParams(max_tokens=20), kv4=True)
    assert got.tokens == want
    # decode_greedy from the first id on, in a cache used before
    cache.reset()
    assert cache.total_len() == 0
    m.forward_seq(prompt, cache)
    ids, ms = m.decode_greedy(want[0], 12, cache)
    assert [int(t) for t in ids] == want[1:13] and ms > 0
    # sampled: the same draws give the same ids
    p = T.GenParams(max_tokens=12, temperature=0.8, top_k=20, top_p=0.9, repetition_penalty=1.1, seed=5)
    assert T.generate(m, prompt, p, kv4=True).tokens == T.generate(m, prompt, p, kv4=True).tokens


def test_f32_caches_beside_4_bit_ones(T, model):
    """Both kinds on one model, steps in turn: neither changes the other."""
    m, tb, w = model
    prompt = [int(t) for t in T.synth_tokens(8, 20, w.vocab_size)]
    alone = m.new_cache(64)
    first = [m.forward_seq(prompt, alone)] + [m.forward_token(t, alone) for t in (3, 5, 9)]
    f32, kv4 = m.new_cache(64), m.new_cache(64, kv4=True)
    second = [m.forward_seq(prompt, f32)]
    other = [m.forward_seq(prompt, kv4)]
    for t in (3, 5, 9):
        other.append(m.forward_token(t, kv4))
        second.append(m.forward_token(t, f32))
    for a, b in zip(first, second):
        np.testing.assert_array_equal(a, b)
    check(m, tb, kv4, prompt + [3, 5, 9], {19 + i: row for i, row in enumerate(other)})


def test_capacity_and_refusals(T, model):
    from tinyminigo_amd._lib import TMG_E_CAPACITY, TMG_E_INVALID, lib
    m, tb, w = model
    cache = m.new_cache(6, kv4=True)
    m.forward_seq([1, 2, 3, 4, 5], cache)
    last = m.forward_token(6, cache)
    with pytest.raises(T.TmgError) as e:
        m.forward_token(7, cache)
    assert e.value.code == TMG_E_CAPACITY
    with pytest.raises(T.TmgError):
        m.forward_seq([1], cache)
    check(m, tb, cache, [1, 2, 3, 4, 5, 6], {5: last})
    with pytest.raises(T.TmgError) as e:
        m.profile_step_floor(1, m.new_cache(64, kv4=True))
    assert e.value.code == TMG_E_INVALID
    h = C.c_void_p()
    assert lib.tmg_cache_new_kv4(m._h, 0, C.byref(h)) == TMG_E_INVALID
    assert lib.tmg_cache_new_kv4(m._h, (1 << 30) + 1, C.byref(h)) == TMG_E_INVALID
    assert lib.tmg_cache_new_kv4(None, 8, C.byref(h)) == TMG_E_INVALID


def test_profile_names_the_attention(T, model):
    m, tb, w = model
    cache = m.new_cache(64, kv4=True)
    m.forward_seq([1, 2, 3], cache)
    kinds = {name: (nbytes, launches) for name, nbytes, ms, launches in m.profile_decode_step(4, cache)}
    c = m.config
    assert "attn_decode" not in kinds and kinds["attn_decode_kv4"][1] == c.num_hidden_layers
    row = 2 * c.num_key_value_heads * (c.head_dim // 2 + R.groups(c.head_dim))
    assert kinds["attn_decode_kv4"][0] == 4 * row + 8 * (c.num_key_value_heads + c.num_attention_heads) * c.head_dim
    assert cache.total_len() == 3


def test_long_session(T):
    """Some thousand positions at the benchmark's head layout: a prompt long
    enough for the prompts' attention, then steps with many runs of keys."""
    from oracle import oracle as O
    from tinyminigo_amd import workloads as W
    w = dataclasses.replace(W.ONE_B, name="kv4-1b-l1", num_hidden_layers=1, vocab_size=512, intermediate_size=256,
                            hidden_size=256, weight_seed=32)
    path = W.ensure_model(w, model_root())
    m = T.Model.load(path)
    tb = Decoder(m.config, O.load_safetensors(path))
    cache = m.new_cache(2400, kv4=True)
    tokens = [int(t) for t in T.synth_tokens(70, 2200, w.vocab_size)]
    row, logits = m.forward_seq(tokens, cache), {}
    logits[2199] = row
    for _ in range(5):
        t = int(np.argmax(row))
        row = m.forward_token(t, cache)
        tokens.append(t)
        logits[len(tokens) - 1] = row
    check(m, tb, cache, tokens, logits)
