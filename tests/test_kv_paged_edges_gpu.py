"""The paged decode engine (PagedKVDecoder) in the calls that its other tests do not make."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def engine(n_heads=4, n_kv=2, d_head=32, d_model=128, n_layers=2):
    from toy_b200 import FromScratch, LlamaConfig, RecipeOptions
    rec = FromScratch()
    rec.realize(LlamaConfig(512, d_model, n_heads, n_kv, d_head, 256, n_layers, 1e4, 1e-5),
                RecipeOptions(t_seq=64, t_batch=1, seed=3))
    return rec.fs_cache


def test_sizes_past_64_bits(cuda):
    """Pools whose bytes pass 2^64 are refused as those that the GPU cannot hold (here 2^64 itself: 0 when cut)."""
    from toy_b200._lib import lib
    eng = engine(n_heads=8, n_kv=8, d_head=128, n_layers=4)
    for n_pages in (1 << 30, 2 ** 31 - 1):
        assert lib().tb2_kv_realize_paged(eng.sess, 32, 1, 0, 1 << 20, n_pages) == -3


def test_many_pages(cuda):
    """More free pages than are put on the stack at a time."""
    from toy_b200.decode import PagedKVDecoder
    eng = engine()
    n = (1 << 20) + 3
    dec = PagedKVDecoder(eng, max_T=8, n_seq=2, n_pages=n, page_size=1, kv_type="q8_0")
    first = dec.decode_step([5, 6])
    assert dec.state()[1] == n - 2
    dec.reset()
    assert dec.state()[1] == n and np.array_equal(dec.decode_step([5, 6]), first)
    dec.close()


def test_generate_again(cuda):
    """A second call starts anew: its continuations are those of a fresh decoder, whatever the sequences held."""
    from toy_b200.decode import KVDecoder, PagedKVDecoder
    eng = engine()
    calls = [([[3, 1, 4], [1, 5]], 6), ([[9, 2, 6, 5], [3]], 5), ([[3, 1, 4], [1, 5]], 6)]
    want = []
    for prompts, n_new in calls:
        want.append([])
        for p in prompts:
            d = KVDecoder(eng, max_T=16, n_seq=1)
            want[-1].append(d.generate(np.asarray([p]), n_new)[0].tolist())
            d.close()
    dec = PagedKVDecoder(eng, max_T=16, n_seq=2, n_pages=8, page_size=4, kv_type="f32")
    for (prompts, n_new), w in zip(calls, want):
        assert dec.generate(prompts, n_new) == w
        assert dec.state()[0].tolist() == [len(p) + n_new - 1 for p in prompts]
        dec.decode_step([7, -1])                    # and what is appended between calls is gone
    dec.close()


def test_generate_refusals(cuda):
    """What a call cannot complete is refused before it changes anything."""
    from toy_b200.decode import PagedKVDecoder
    dec = PagedKVDecoder(engine(), max_T=12, n_seq=2, n_pages=5, page_size=4, kv_type="f32")
    dec.decode_step([1, 2])
    dec.decode_step([3, -1])
    held = dec.state()[0].tolist()
    for prompts, n_new, error in (([[1] * 8, [1]], 6, ValueError), ([[1] * 8, [1] * 8], 5, MemoryError),
                                  ([[1, -1], [1]], 2, ValueError), ([[1, 512], [1]], 2, ValueError),
                                  ([[1], []], 2, ValueError), ([[1]], 2, ValueError)):
        with pytest.raises(error):
            dec.generate(prompts, n_new)
        assert dec.state()[0].tolist() == held == [2, 1] and dec.state()[1] == 3
    assert dec.generate([[1], [2]], 0) == [[], []] and dec.state()[0].tolist() == held
    assert [len(x) for x in dec.generate([[1] * 8, [1] * 4], 5)] == [5, 5]    # 3 + 2 pages: just enough
    dec.close()


def test_release_refusals(cuda):
    """Sequences that are none are refused; an empty list and repeats are not."""
    from toy_b200.decode import PagedKVDecoder
    dec = PagedKVDecoder(engine(), max_T=12, n_seq=3, n_pages=6, page_size=4, kv_type="f32")
    dec.decode_step([1, 2, 3])
    for bad in ([-1], [3], [0, -3], [1, 100]):
        with pytest.raises(ValueError):
            dec.release(bad)
        assert dec.state()[0].tolist() == [1, 1, 1]
    dec.release([])
    dec.release([1, 1])
    assert dec.state()[0].tolist() == [1, 0, 1] and dec.state()[1] == 4
    dec.close()


def test_sizes_past_32_bits(cuda):
    """Sizes that the entry point's 32 bits would cut."""
    from toy_b200.decode import PagedKVDecoder
    eng = engine()
    for kw in (dict(n_pages=2 ** 32 + 4), dict(max_T=2 ** 32 + 4), dict(page_size=2 ** 32 + 4)):
        with pytest.raises(ValueError):
            PagedKVDecoder(eng, **{**dict(max_T=8, n_seq=1, n_pages=4, page_size=4), **kw})
