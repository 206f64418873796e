"""Decode over a paged cache (tb2_kv_*_paged through PagedKVDecoder) against the
oracle's full-sequence forward: sequences of unlike lengths that start, pause,
finish and reuse pages, the logits after each token within the bounds of the
contiguous decoder's tests (f32 cache 1e-4 relative L2 per row; Q8_0, f16 and
bf16 caches against the oracle with the same rounding of K and V, 1e-3 at the
median and 1e-2 per row, since a value on a rounding boundary may land on either
side)."""
import numpy as np
import pytest

from oracle import oracle as O

pytestmark = pytest.mark.gpu


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return np.linalg.norm(a - b) / np.linalg.norm(b)


def tiny(n_heads=4, n_kv=2, d_head=32):
    from toy_b200 import LlamaConfig
    oc = O.LlamaCfg(vocab=512, d_model=128, n_heads=n_heads, n_kv=n_kv, d_head=d_head, d_ff=256, n_layers=2,
                    rope_base=1e4)
    return oc, LlamaConfig(512, 128, n_heads, n_kv, d_head, 256, 2, 1e4, 1e-5)


def base_model(mode, oc, gc, seed):
    from toy_b200 import FromScratch, LoRA, LoraOptions, RecipeOptions
    if mode == "q8":
        rec = LoRA()
        targets = ("q", "v", "o")
        rec.realize(gc, 8, RecipeOptions(t_seq=64, t_batch=1, seed=seed), LoraOptions(rank=8, targets=targets))
        mdl = O.qlora_model(oc, O.LoraCfg(rank=8, alpha=16.0, targets=targets), seed=seed)
        rng = np.random.default_rng(seed)
        for k in mdl.trainable:
            if k.endswith(".lora_b"):
                v = (rng.standard_normal(mdl.params[k].shape) * 0.05).astype(np.float32)
                mdl.params[k] = v
                rec.lora_cache.set_param(k, v)
        return rec.lora_cache, mdl
    rec = FromScratch()
    rec.realize(gc, RecipeOptions(t_seq=64, t_batch=1, seed=seed))
    return rec.fs_cache, O.full_ft_model(oc, seed=seed)


def rounded(cache, monkeypatch):
    """The oracle's K / V round trip for this cache type; whether it is used."""
    if cache in ("f16", "bf16"):
        import torch
        t = {"f16": torch.float16, "bf16": torch.bfloat16}[cache]
        monkeypatch.setattr(O, "q8_0_roundtrip",
                            lambda x: torch.from_numpy(np.ascontiguousarray(x)).float().to(t).float().numpy())
    return cache != "f32"


def rows_of(mdl, oc, ids, kv_q8):
    n = len(ids)
    _, _, ref = O.forward_backward(mdl, np.asarray(ids), O.positions(n, 1), O.next_token_labels(np.asarray(ids), n, 1,
                                                                                                 oc.vocab),
                                   n, 1, want_grads=False, kv_q8=kv_q8)
    return ref.reshape(n, -1)


@pytest.mark.parametrize("mode", ["q8", "f32"])
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("heads,page", [((4, 2, 32), 16), ((9, 3, 64), 5)])
def test_ragged_decode(cuda, mode, cache, heads, page, monkeypatch):
    from toy_b200.decode import PagedKVDecoder
    from toy_b200._lib import lib
    oc, gc = tiny(*heads)
    eng, mdl = base_model(mode, oc, gc, 3)
    kv_q8 = rounded(cache, monkeypatch)
    lengths, n_seq = [40, 1, 17, 33], 4
    ids = [O.token_ids(20 + b, n, oc.vocab) for b, n in enumerate(lengths)]
    pages = sum(-(-n // page) for n in lengths)
    dec = PagedKVDecoder(eng, max_T=40, n_seq=n_seq, n_pages=pages, page_size=page, kv_type=cache)
    fed, got = [0] * n_seq, [[] for _ in range(n_seq)]
    rng = np.random.default_rng(7)
    while any(fed[b] < lengths[b] for b in range(n_seq)):
        # sequences advance at their own pace
        on = [fed[b] < lengths[b] and rng.random() < (0.9, 0.5, 0.6, 0.8)[b] for b in range(n_seq)]
        if not any(on):
            continue
        logits = dec.decode_step([ids[b][fed[b]] if on[b] else -1 for b in range(n_seq)])
        for b in range(n_seq):
            if on[b]:
                got[b].append(logits[b])
                fed[b] += 1
    lens, free = dec.state()
    assert lens.tolist() == lengths and free == 0
    errs = []
    for b in range(n_seq):
        ref = rows_of(mdl, oc, ids[b], kv_q8)
        errs += [rel(got[b][t], ref[t]) for t in range(lengths[b])]
    errs = np.array(errs)
    if kv_q8:
        assert float(np.median(errs)) < 1e-3 and float(errs.max()) < 1e-2, (float(np.median(errs)), float(errs.max()))
    else:
        assert float(errs.max()) < 1e-4, float(errs.max())
    dec.release([2])
    lens, free = dec.state()
    assert lens.tolist() == [40, 1, 0, 33] and free == -(-17 // page)
    # the freed pages serve another sequence, whose logits are the same as the first one's
    for t in range(17):
        again = dec.decode_step([-1, -1, ids[2][t], -1])[2]
        assert np.array_equal(again, got[2][t]) or rel(again, got[2][t]) < 1e-5
    dec.close()
    assert lib().tb2_device_error() == 0


def test_no_room_and_reset(cuda):
    from toy_b200.decode import KVDecoder, PagedKVDecoder
    from toy_b200._lib import lib
    oc, gc = tiny()
    eng, _ = base_model("q8", oc, gc, 3)
    dec = PagedKVDecoder(eng, max_T=12, n_seq=3, n_pages=4, page_size=4, kv_type="bf16")
    first = dec.decode_step([5, 6, 7])
    for t in range(3):
        dec.decode_step([1, 2, 3])
    dec.decode_step([9, -1, -1])                    # the fourth and last page
    with pytest.raises(MemoryError):
        dec.decode_step([1, 2, -1])                 # sequence 1 needs a fifth: sequence 0 gets no token either
    lens, free = dec.state()
    assert lens.tolist() == [5, 4, 4] and free == 0
    dec.decode_step([1, -1, -1])                    # its open page still has room
    dec.release([1, 2])
    assert dec.state()[1] == 2
    for t in range(6):
        dec.decode_step([2, -1, -1])
    with pytest.raises(RuntimeError):
        dec.decode_step([2, -1, -1])                # past max_T
    for bad in ([-1, -1, -1], [oc.vocab, 0, 0], [-2, 0, 0]):
        with pytest.raises(RuntimeError):
            dec.decode_step(bad)
    dec.reset()
    assert dec.state()[0].tolist() == [0, 0, 0] and dec.state()[1] == 4
    assert np.array_equal(dec.decode_step([5, 6, 7]), first)
    # one decode engine of either kind per session, each with its own calls
    L, s = lib(), eng.sess
    assert L.tb2_kv_realize_paged(s, 12, 3, 30, 4, 4) == -2 and L.tb2_kv_realize(s, 12, 3, 0) == -2
    toks = (np.zeros(3, np.int64), np.zeros(3, np.int64))
    import ctypes as C
    ll = [t.ctypes.data_as(C.POINTER(C.c_longlong)) for t in toks]
    assert L.tb2_kv_decode(s, ll[0], ll[1], 3, None) == -2
    assert L.tb2_kv_run(s, 1, C.byref(C.c_float())) == -2
    dec.close()
    assert L.tb2_kv_decode_paged(s, ll[0], 3, None) == -2
    for bad in ((0, 3, 30, 4, 4), (12, 3, 2, 4, 4), (12, 9, 30, 4, 4), (12, 3, 30, 0, 4), (12, 3, 30, 4, 0),
                (1 << 30, 3, 30, 4, 4)):
        assert L.tb2_kv_realize_paged(s, *bad) == -1
    other = KVDecoder(eng, max_T=12, n_seq=3)
    assert L.tb2_kv_decode_paged(s, ll[0], 3, None) == -2
    assert L.tb2_kv_release(s, (C.c_int * 3)(), 3) == -2
    other.close()


def test_generate_matches_contiguous(cuda):
    """Greedy continuations of three prompts of unlike lengths: the contiguous decoder's, sequence by sequence."""
    from toy_b200.decode import KVDecoder, PagedKVDecoder
    oc, gc = tiny()
    eng, _ = base_model("q8", oc, gc, 5)
    prompts = [O.token_ids(b, n, oc.vocab) for b, n in ((1, 9), (2, 3), (4, 20))]
    want = []
    for p in prompts:
        d = KVDecoder(eng, max_T=64, n_seq=1)
        want.append(d.generate(np.asarray(p)[None, :], 6)[0].tolist())
        d.close()
    dec = PagedKVDecoder(eng, max_T=64, n_seq=3, n_pages=20, page_size=8, kv_type="f32")
    assert dec.generate(prompts, 6) == want
    dec.close()


def family(name):
    from toy_b200 import LlamaConfig
    if name == "bias":
        return (O.LlamaCfg(vocab=512, d_model=256, n_heads=4, n_kv=2, d_head=128, d_ff=640, n_layers=2, rope_base=1e6,
                           rms_eps=1e-6, qkv_bias=True),
                LlamaConfig(512, 256, 4, 2, 128, 640, 2, 1e6, 1e-6, qkv_bias=True))
    ff = O.llama3_freq_factors(64, 5.0e5, 8192, 32.0, 1.0, 4.0)
    return (O.LlamaCfg(vocab=640, d_model=256, n_heads=10, n_kv=1, d_head=64, d_ff=512, n_layers=2, rope_base=5.0e5,
                       rope_freq_factors=ff),
            LlamaConfig(640, 256, 10, 1, 64, 512, 2, 5.0e5, 1e-5, rope_freq_factors=list(ff)))


@pytest.mark.parametrize("name", ["bias", "freq_factors"])
@pytest.mark.parametrize("mode", ["q8", "f32"])
@pytest.mark.parametrize("cache", ["f32", "q8_0"])
def test_families(cuda, name, mode, cache, monkeypatch):
    """q, k and v biases; scaled RoPE frequencies with one key head for ten query heads: 24 tokens of a sequence beside
    one that starts 9 tokens later, against the oracle's rows."""
    from toy_b200.decode import PagedKVDecoder
    from toy_b200._lib import lib
    oc, gc = family(name)
    eng, mdl = base_model(mode, oc, gc, 3)
    kv_q8 = rounded(cache, monkeypatch)
    ids = O.token_ids(31, 24, oc.vocab)
    dec = PagedKVDecoder(eng, max_T=24, n_seq=2, n_pages=10, page_size=7, kv_type=cache)
    late, got = 9, [[], []]
    for t in range(24 + late):
        toks = [ids[t] if t < 24 else -1, ids[t - late] if t >= late else -1]
        logits = dec.decode_step(toks)
        for b in range(2):
            if toks[b] >= 0:
                got[b].append(logits[b])
    dec.close()
    ref = rows_of(mdl, oc, ids, kv_q8)
    errs = np.array([rel(got[b][t], ref[t]) for b in range(2) for t in range(24)])
    if kv_q8:
        assert float(np.median(errs)) < 1e-3 and float(errs.max()) < 1e-2, (float(np.median(errs)), float(errs.max()))
    else:
        assert float(errs.max()) < 1e-4, float(errs.max())
    assert lib().tb2_device_error() == 0


def test_smollm2_shape(cuda):
    """The SmolLM2-135M shape, 16 sequences of unlike lengths, against single-sequence oracle rows."""
    from toy_b200 import LlamaConfig
    from toy_b200.decode import PagedKVDecoder
    oc, gc = O.smollm2_135m(), LlamaConfig.smollm2_135m()
    eng, mdl = base_model("q8", oc, gc, 42)
    n_seq = 16
    lengths = [3 + 2 * b for b in range(n_seq)]
    ids = [O.token_ids(60 + b, n, oc.vocab) for b, n in enumerate(lengths)]
    dec = PagedKVDecoder(eng, max_T=64, n_seq=n_seq, n_pages=64, page_size=16, kv_type="f32")
    got = [None] * n_seq
    for t in range(max(lengths)):
        toks = [ids[b][t] if t < lengths[b] else -1 for b in range(n_seq)]
        logits = dec.decode_step(toks)
        for b in range(n_seq):
            if t == lengths[b] - 1:
                got[b] = logits[b].copy()
    for b in (0, 7, 15):
        assert rel(got[b], rows_of(mdl, oc, ids[b], False)[-1]) < 1e-4
    dec.close()
