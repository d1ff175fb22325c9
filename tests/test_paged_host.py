"""The host side of the paged cache's and draft verification's Python layer, on
the CPU: where memory comes from, first calls of several threads, arguments that
do not fit the C types."""
import contextlib
import sys

import pytest


@pytest.fixture
def pk():
    from cudalm_w4a16 import paged_kv

    return paged_kv


@pytest.mark.parametrize("stream,want", [(0, ("default", 0)), (0x5500, ("external", 0x5500)), (None, None),
                                         ("a stream object", "a stream object")])
def test_memory_is_of_the_stream_that_the_call_runs_on(pk, monkeypatch, stream, want):
    """Handle 0 is the default stream, which torch gives by another name than streams of a handle
    (0 there means no handle, and a stream of torch's pool)."""
    import torch

    current = [None]

    @contextlib.contextmanager
    def run_on(s):
        current[0] = s
        yield
        current[0] = None

    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device=None: ("external", handle))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: ("default", getattr(device, "index", device)))
    monkeypatch.setattr(torch.cuda, "stream", run_on)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: current[0])
    assert pk._empty((3,), torch.uint8, 0, stream) == want


def test_rows_of_one_token_are_equally_spaced(pk):
    """The strides of dimensions of one entry say nothing: one token per sequence out of a longer tensor
    has the batch's stride, a single one any."""
    import torch

    like = torch.empty(1, 2, 16, 128, dtype=torch.bfloat16)
    x = torch.empty(3, 5, 8, 128, dtype=torch.bfloat16)
    rows = lambda t, cols: pk._rows(t, cols, None, like, -1, "q")  # noqa: E731
    assert rows(x[:, -1:], 2) == (5 * 8 * 128, 128)
    assert rows(x[:, -1], 1) == (5 * 8 * 128, 128)
    assert rows(x, 2) == (8 * 128, 128)
    assert rows(x[:1, 1:3], 2) == (8 * 128, 128)
    assert rows(x[:, :, :1], 2) == (8 * 128, 0)
    odd = torch.empty(9, 8, 132, dtype=torch.bfloat16)[:, :, :128]
    assert rows(odd.as_strided((1, 8, 128), (3, 128, 1)), 1) == (0, 128)
    assert rows(odd.as_strided((1, 1, 1, 128), (3, 5, 7, 1)), 2) == (0, 0)
    with pytest.raises(ValueError):
        rows(x[:, 1:3], 2)  # two tokens of each of five
    with pytest.raises(ValueError):
        rows(x[:, -1:].transpose(2, 3).contiguous().transpose(2, 3), 2)  # a head's elements apart


def test_one_row_of_probabilities_per_sequence():
    import torch

    from cudalm_w4a16 import draft

    probs = lambda t, rows, V: draft._probs(t, t.shape[0], rows, V, torch.float32, -1, "target")  # noqa: E731
    x = torch.empty(3, 5, 100)
    assert probs(x[:, :1], 1, 100) == 500
    assert probs(x[:, :1, :90], 1, 90) == 500
    assert probs(x, 5, 100) == 100
    assert probs(x[:1, 1:3], 2, 100) == 100
    assert probs(x[:1, 1:2], 1, 100) >= 100
    assert probs(x.as_strided((1, 1, 100), (1, 3, 1)), 1, 100) >= 100
    assert probs(x.as_strided((3, 5, 1), (500, 100, 2)), 5, 1) == 100  # a vocabulary of one
    with pytest.raises(ValueError):
        probs(x[:, 1:3], 2, 100)
    with pytest.raises(ValueError):
        probs(x[:, :1, ::2], 1, 50)


BIG = [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1, 10 ** 30]


@pytest.mark.parametrize("value", BIG)
@pytest.mark.parametrize("name", ["window", "sinks", "max_len"])
def test_options_past_32_bits_of_a_query_are_refused(pk, name, value):
    import torch

    q = torch.empty(3, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=name):
        pk._query(q, q, 1024, 128, None, **{**dict(window=0, sinks=0, max_len=None), name: value})


@pytest.mark.parametrize("value", BIG)
@pytest.mark.parametrize("name", ["keep", "sinks", "recent", "max_len"])
def test_options_past_32_bits_of_an_eviction_are_refused(pk, name, value):
    """ctypes would pass their lower 32 bits."""
    import torch

    k, v, w = pk.empty_cache(4, 16, 2, 128, torch.bfloat16, device="cpu", weights=True)
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match=name):
        pk.evict(k, v, tables, lens, w, tables, **{"keep": 3, name: value})


def test_types_are_all_there_once_the_first_is_seen(pk, monkeypatch):
    """A second thread's first call goes on as soon as _types is set."""
    import torch

    seen = []

    class Torch:
        def __getattr__(self, name):
            seen.append((name, pk._types))
            return getattr(torch, name)

    monkeypatch.setitem(sys.modules, "torch", Torch())
    monkeypatch.setattr(pk, "_types", None)
    pk._load_types()
    assert {"bfloat16", "float16", "int32", "float32"} <= {n for n, _ in seen}
    assert all(types is None for _, types in seen)
    assert pk._types == {torch.bfloat16: pk.BF16, torch.float16: pk.F16} and pk._int32_type is torch.int32


def test_decode_of_tiles_that_31_bits_do_not_number_is_refused(pk, w4):
    """The last workgroup's range of tiles ends past the last tile: there has to be room for it."""
    import ctypes

    lib, fake = w4.lib(), 0x100000
    q = pk.Query(q=fake, out=fake, token_stride=1024, head_stride=128, heads=8, scale=0.1)

    def served(batch, max_pages):
        kv = pk.KV(k=fake, v=fake, tables=fake, lens=fake, num_pages=10, page_size=16, kv_heads=2, head_dim=128,
                   batch=batch, max_pages=max_pages)
        args = (ctypes.byref(kv), ctypes.byref(q), 1, 0)
        if lib.cudalm_paged_decode_workspace_bytes(*args):
            return True
        assert lib.cudalm_paged_decode(*args, fake, 1 << 40, None) == w4.ERANGE
        return False

    assert not served(33, 2 ** 26) and not served(32, 2 ** 26)
    assert not served(32, 2 ** 26 - 4)  # 64 x (2^25 - 2) tiles of 32 tokens
    assert served(31, 2 ** 26) and served(62, 2 ** 25)
