"""The paged operators' and the sampler's checks, which come before any CUDA call: the addresses here
are made up, and no GPU is needed."""

import contextlib
import ctypes
import gc
import threading
import weakref

import pytest
import torch

from qwenscriber_b200 import paged, paged_decoder, sampling
from qwenscriber_b200 import runtime as rt

A = 1 << 20  # aligned to everything


def cache(**kw):
    d = dict(k_scales=A, k_codes=A, v_scales=A, v_codes=A, pages=10, page_size=16, kv_heads=2, head_dim=128)
    d.update(kw)
    return rt.PagedCacheDesc(*d.values())


def batch(**kw):
    d = dict(query_starts=A, context_lens=A, page_table=A, sequences=2, tokens=2, table_stride=5, max_query=1, max_context=80,
             reserved=0)
    d.update(kw)
    return rt.PagedBatchDesc(*d.values())


def attention(c, b, fmt=0, q=A, q_stride=512, heads=4, out=A, out_stride=512, work=A, size=1 << 40):
    return rt.lib().qwc_op_paged_attention(ctypes.addressof(c), ctypes.addressof(b), fmt, q, q_stride, heads, out, out_stride, work,
                                           size, None)


def append(c, b, fmt=0, q=A, q_stride=1024, k=A, k_stride=1024, v=A, v_stride=1024, heads=4, qn=A, kn=A, cos=A, sin=A, out=A,
           out_stride=1024):
    return rt.lib().qwc_op_paged_append(ctypes.addressof(c), ctypes.addressof(b), fmt, q, q_stride, k, k_stride, v, v_stride, heads,
                                        qn, kn, 1e-6, cos, sin, 100, out, out_stride, None)


def read(c, b, fmt=0, k=A, k_stride=256, v=A, v_stride=256):
    return rt.lib().qwc_op_paged_read(ctypes.addressof(c), ctypes.addressof(b), fmt, k, k_stride, v, v_stride, None)


INVALID, UNSUPPORTED, SHAPE, LIMIT = (rt.STATUS_CODE[n] for n in ("invalid_argument", "unsupported", "shape_mismatch", "limit_exceeded"))

POOL = [
    (dict(k_scales=None), {}, INVALID), (dict(v_codes=A + 8), {}, INVALID), (dict(k_codes=A + 1), {}, INVALID),
    ({}, dict(page_table=None), INVALID), ({}, dict(query_starts=A + 2), INVALID),
    (dict(head_dim=96), {}, UNSUPPORTED), (dict(head_dim=256), {}, UNSUPPORTED), (dict(head_dim=0), {}, UNSUPPORTED),
    (dict(kv_heads=0), {}, SHAPE), (dict(page_size=0), {}, SHAPE), (dict(pages=0), {}, SHAPE),
    ({}, dict(max_context=81), SHAPE), (dict(pages=1 << 31, page_size=16), {}, LIMIT), ({}, dict(sequences=70000), LIMIT),
]


@pytest.mark.parametrize("call", [attention, append, read])
@pytest.mark.parametrize("c,b,status", POOL)
def test_descriptors_are_checked(cuda_lib, call, c, b, status):
    assert call(cache(**c), batch(**b)) == status


def test_null_descriptors(cuda_lib):
    L = rt.lib()
    c = ctypes.addressof(cache())
    assert L.qwc_op_paged_read(None, None, 0, A, 256, A, 256, None) == INVALID
    assert L.qwc_op_paged_read(c, None, 0, A, 256, A, 256, None) == INVALID
    assert L.qwc_op_paged_attention_workspace(c, None, 0, 4, None) == INVALID


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=16), UNSUPPORTED), (dict(q=None), INVALID), (dict(q=A + 4), INVALID), (dict(out=A + 8), INVALID),
    (dict(q_stride=513), INVALID), (dict(fmt=2, q_stride=516), INVALID), (dict(q_stride=256), SHAPE), (dict(out_stride=508), SHAPE),
    (dict(heads=0), SHAPE), (dict(heads=5), SHAPE), (dict(work=None), INVALID), (dict(work=A + 4), INVALID), (dict(size=0), LIMIT),
])
def test_attention_arguments(cuda_lib, kw, status):
    assert attention(cache(), batch(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=3), UNSUPPORTED), (dict(k=None), INVALID), (dict(v=A + 4), INVALID), (dict(cos=None), INVALID), (dict(sin=A + 4), INVALID),
    (dict(qn=A + 4), INVALID), (dict(kn=A + 8), INVALID), (dict(k_stride=252), SHAPE), (dict(v_stride=1022), INVALID),
    (dict(heads=3), SHAPE), (dict(out=None), INVALID),
])
def test_append_arguments(cuda_lib, kw, status):
    assert append(cache(), batch(), **kw) == status


@pytest.mark.parametrize("kw,status", [(dict(fmt=18), UNSUPPORTED), (dict(k=None), INVALID), (dict(v=A + 2), INVALID),
                                       (dict(k_stride=128), SHAPE), (dict(fmt=1, v_stride=260), INVALID)])
def test_read_arguments(cuda_lib, kw, status):
    assert read(cache(), batch(), **kw) == status


def test_nothing_to_do_launches_nothing(cuda_lib):
    # No tokens, or no sequences: ok without a device.
    for b in (batch(tokens=0), batch(max_query=0), batch(sequences=0)):
        assert attention(cache(), b) == 0 and append(cache(), b) == 0 and read(cache(), b) == 0


def test_workspace_is_bounded_by_the_batch(cuda_lib):
    def need(b, fmt=0, heads=4):
        n = ctypes.c_uint64(0)
        assert rt.lib().qwc_op_paged_attention_workspace(ctypes.addressof(cache()), ctypes.addressof(b), fmt, heads, ctypes.byref(n)) == 0
        return n.value

    assert 0 < need(batch()) <= need(batch(sequences=64, tokens=64))
    assert need(batch(sequences=64, tokens=64 * 512, max_query=512, max_context=80)) < 1 << 30


@pytest.mark.parametrize("kw,status", [
    (dict(fmt=16), UNSUPPORTED), (dict(logits=None), INVALID), (dict(uniforms=None), INVALID), (dict(out=None), INVALID),
    (dict(vocab=0), INVALID), (dict(logits=A + 2), INVALID), (dict(fmt=1, logits=A + 1), INVALID), (dict(top_k=A + 2), INVALID),
    (dict(stride=99), SHAPE), (dict(vocab=rt.SAMPLE_MAX_VOCAB + 1, stride=1 << 21), LIMIT),
])
def test_sample_arguments(cuda_lib, kw, status):
    d = dict(fmt=0, logits=A, stride=100, rows=2, vocab=100, temperature=A, top_k=A, top_p=A, min_p=A, uniforms=A, out=A, logprobs=A)
    d.update(kw)
    assert rt.lib().qwc_op_sample(*d.values(), None) == status


def test_sample_of_no_rows(cuda_lib):
    assert rt.lib().qwc_op_sample(0, A, 100, 0, 100, None, None, None, None, A, A, None, None) == 0


def host_batch(table, max_context):
    n = table.shape[0]
    ints = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    return paged.PagedBatch(ints(range(n + 1)), ints([1] * n), table, tokens=n, max_query=1, max_context=max_context)


@pytest.mark.parametrize("view,entries", [
    (lambda t: t, 100), (lambda t: t[:, 96:], 4), (lambda t: t[:, 3:8], 5), (lambda t: t[:1, 90:], 10), (lambda t: t[:1, :7].expand(3, 7), 7),
    (lambda t: t[1:2, 40:41].expand(3, 1), 1),
])
def test_a_table_is_as_long_as_its_columns(cuda_lib, view, entries):
    # Not as its rows are apart: an entry past a view's columns is another sequence's, or past the storage.
    table = view(torch.zeros(3, 100, dtype=torch.int32))
    pool = paged.PagedCache.zeros(10, 16, 2, 128, device="cpu")
    assert paged.workspace_bytes(pool, host_batch(table, 16 * entries), 4, 0) > 0
    with pytest.raises(rt.QwcError) as e:
        paged.workspace_bytes(pool, host_batch(table, 16 * entries + 1), 4, 0)
    assert e.value.name == "shape_mismatch"


@pytest.mark.parametrize("b,status", [
    (dict(table_stride=100, max_context=81), SHAPE), (dict(table_stride=100, max_context=80), 0), (dict(table_stride=0, max_context=80), 0),
    (dict(table_stride=3, max_context=81), SHAPE),
])
def test_entries_bound_the_context(cuda_lib, b, status):
    n = ctypes.c_uint64(0)
    d = batch(**b)
    d.table_entries = 5
    assert rt.lib().qwc_op_paged_attention_workspace(ctypes.addressof(cache()), ctypes.addressof(d), 0, 4, ctypes.byref(n)) == status


class Stub:
    """A tensor of a device that is not there."""

    def __init__(self, *shape, dtype=torch.float32, device="cuda:1"):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, torch.device(device)

    dim = lambda self: len(self.shape)  # noqa: E731
    numel = lambda self: self.shape.numel()  # noqa: E731
    data_ptr = lambda self: A  # noqa: E731
    is_contiguous = lambda self: True  # noqa: E731

    def stride(self, i=None):
        strides = [self.shape[j + 1:].numel() for j in range(self.dim())]
        return strides if i is None else strides[i]


def stub_calls(device):
    """Each call of the package on tensors of `device`."""
    t = lambda *shape, dtype=torch.float32: Stub(*shape, dtype=dtype, device=device)  # noqa: E731
    planes = [t(160, 4, dtype=torch.float16), t(160, 256, dtype=torch.uint8)] * 2
    pool = paged.PagedCache(*planes, page_size=16, kv_heads=2, head_dim=128)
    i32 = torch.int32
    b = paged.PagedBatch(t(3, dtype=i32), t(2, dtype=i32), t(2, 5, dtype=i32), tokens=2, max_query=1, max_context=80)
    q, kv, table = t(2, 4, 128), t(2, 2, 128), t(100, 64)
    return {
        "append": lambda: paged.append(pool, b, q, kv, kv, table, table, q_out=q),
        "attention": lambda: paged.attention(pool, b, q, q, t(1 << 30, dtype=torch.uint8)),
        "read": lambda: paged.read(pool, b, torch.float32, kv, kv),
        "sample": lambda: sampling.sample(t(2, 100), t(2)),
    }


CALLS = ["append", "attention", "read", "sample"]


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("current", [0, 1, 2])
def test_launches_go_to_the_tensors_device(monkeypatch, name, current):
    at, launched, entered = [current], [], []

    class Current:
        def __init__(self, device):
            self.index = device

        def __enter__(self):
            entered.append(self.index)
            self.before, at[0] = at[0], self.index

        def __exit__(self, *a):
            at[0] = self.before

    class Lib:
        def __getattr__(self, name):
            return lambda *a: launched.append((name, at[0], a[-1])) or 0

    calls = stub_calls("cuda:1")
    monkeypatch.setattr(paged, "_current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", Current)
    monkeypatch.setattr(torch, "empty", lambda *shape, dtype, device: Stub(*shape, dtype=dtype, device=device))
    for module in (paged, sampling):
        monkeypatch.setattr(module, "lib", lambda: Lib())
        monkeypatch.setattr(module, "current_stream", lambda device: 1000 + device.index)
    calls[name]()
    assert [c[1:] for c in launched] == [(1, 1001)]
    assert entered == ([] if current == 1 else [1]) and at[0] == current


@pytest.mark.parametrize("name", CALLS)
def test_host_memory_is_refused(monkeypatch, name):
    def launched():
        raise AssertionError("a kernel was given host memory")

    for module in (paged, sampling):
        monkeypatch.setattr(module, "lib", launched)
    with pytest.raises(rt.QwcError) as e:
        stub_calls("cpu")[name]()
    assert e.value.name == "invalid_argument"


def test_an_operator_of_the_decoder_goes_to_its_device(monkeypatch):
    at, launched = [0], []

    @contextlib.contextmanager
    def current(index):
        before, at[0] = at[0], index
        yield
        at[0] = before

    class Lib:
        qwc_op_silu_mul = staticmethod(lambda *a: launched.append((at[0], a[-1])) or 0)

    monkeypatch.setattr(paged, "_current_device", lambda: at[0])
    monkeypatch.setattr(torch.cuda, "device", current)
    monkeypatch.setattr(paged_decoder, "lib", Lib)
    monkeypatch.setattr(paged, "current_stream", lambda device: 1000 + device.index)
    d = object.__new__(paged_decoder.PagedDecoder)
    d.device = torch.device("cuda:1")
    d._call("qwc_op_silu_mul", A, A, 4, A)
    assert launched == [(1, 1001)] and at[0] == 0


def test_a_workspace_lives_until_the_launch(cuda_lib, monkeypatch):
    # Another thread on the stream puts a larger buffer in the place of the one that a call has looked up.
    born, alive = [], []

    def new(need, device):
        buffer = torch.zeros(need, dtype=torch.uint8)
        born.append((buffer.data_ptr(), weakref.ref(buffer)))
        return buffer

    class Lib:
        @staticmethod
        def qwc_op_paged_attention_workspace(cache, batch, fmt, heads, n):
            return rt.lib().qwc_op_paged_attention_workspace(cache, batch, fmt, heads, n)

        @staticmethod
        def qwc_op_paged_attention(*a):
            thread = threading.Thread(target=paged._workspace, args=(pool, a[9] + 4096, 1001))
            thread.start()
            thread.join()
            gc.collect()
            alive.extend(ref() is not None for address, ref in born if address == a[8])
            return 0

    monkeypatch.setattr(paged, "_current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged, "current_stream", lambda device: 1000 + device.index)
    monkeypatch.setattr(paged, "_new_workspace", new)
    monkeypatch.setattr(paged, "_workspaces", {})
    monkeypatch.setattr(paged, "lib", lambda: Lib)
    t = lambda *shape, dtype=torch.float32: Stub(*shape, dtype=dtype)  # noqa: E731
    pool = paged.PagedCache(*[t(160, 4, dtype=torch.float16), t(160, 256, dtype=torch.uint8)] * 2, page_size=16, kv_heads=2, head_dim=128)
    b = paged.PagedBatch(t(3, dtype=torch.int32), t(2, dtype=torch.int32), t(2, 5, dtype=torch.int32), tokens=2, max_query=1, max_context=80)
    q = t(2, 4, 128)
    for _ in range(3):
        paged.attention(pool, b, q, q)
    assert len(alive) == 3 and all(alive)
    gc.collect()
    assert sum(ref() is not None for _, ref in born) == 1  # the stream keeps the largest alone


@pytest.mark.parametrize("device", [None, torch.device("cuda"), torch.device("cuda:1")])
def test_a_wait_that_ran_out_is_found_by_any_name_of_the_device(monkeypatch, device):
    buffer = torch.zeros(rt.PAGED_WORKSPACE_HEAD + 64, dtype=torch.uint8)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    monkeypatch.setattr(paged, "current_stream", lambda d: 1000 + (1 if d.index is None else d.index))
    monkeypatch.setattr(paged, "_workspaces", {(1, 1001): (buffer.data_ptr(), buffer.numel(), buffer)})
    paged.check_waits(device=device)
    buffer[0], buffer[400] = 3, 7
    with pytest.raises(rt.QwcError) as e:
        paged.check_waits(device=device)
    assert e.value.name == "invalid_state" and not buffer.any()
    paged.check_waits(device=device)


def test_a_larger_workspace_still_tells_of_a_wait_that_ran_out(monkeypatch):
    pool = paged.PagedCache(*[Stub(160, 4, dtype=torch.float16), Stub(160, 256, dtype=torch.uint8)] * 2, page_size=16, kv_heads=2, head_dim=128)
    monkeypatch.setattr(paged, "_current_device", lambda: 1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged, "current_stream", lambda device: 1000 + device.index)
    monkeypatch.setattr(paged, "_new_workspace", lambda need, device: torch.zeros(need, dtype=torch.uint8))
    monkeypatch.setattr(paged, "_workspaces", {})
    held = paged._workspace(pool, 40000, 1001)[2]
    held[1] = 2  # the kernel's error word
    assert paged._workspace(pool, 50000, 1001)[1] == 50000
    with pytest.raises(rt.QwcError) as e:
        paged.check_waits(device=torch.device("cuda:1"))
    assert e.value.name == "invalid_state"
    paged.check_waits(device=torch.device("cuda:1"))


def test_stretches_of_more_places_than_are_counted_in_31_bits(cuda_lib):
    # A tile of one step takes four places: 65535 sequences of 1024 kv heads and 1211 tiles each are 2.2e9 places to a CTA.
    b = batch(sequences=65535, tokens=(1 << 31) - 1, max_query=310000, max_context=16, table_stride=1)
    assert attention(cache(kv_heads=1024, head_dim=64), b, q_stride=1024 * 64, heads=1024, out_stride=1024 * 64) == LIMIT


def test_a_batch_of_no_sequences(cuda_lib):
    # Its arrays have no elements, so no addresses.
    b = batch(sequences=0, tokens=0, query_starts=None, context_lens=None, page_table=None, table_stride=0)
    for max_context in (0, 80):
        b.max_context = max_context
        assert attention(cache(), b) == 0 and append(cache(), b) == 0 and read(cache(), b) == 0


def test_a_single_token_may_lie_in_a_row_of_any_width(monkeypatch):
    # Nothing is a row's stride away from the only row.
    class Row(Stub):
        def stride(self, i=None):
            strides = [1001, self.shape[2], 1]
            return strides if i is None else strides[i]

    b = paged.PagedBatch(Stub(2, dtype=torch.int32), Stub(1, dtype=torch.int32), Stub(1, 5, dtype=torch.int32), tokens=1, max_query=1, max_context=80)
    assert paged._rows(Row(1, 4, 128), b, 4, 128, "test") == 512
