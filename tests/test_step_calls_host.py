"""What the Python calls of a step hand to the library and what they refuse before, on host tensors: the library is a list of the calls it gets."""

import contextlib

import pytest
import torch

from turboquant_amd import _ffi
from turboquant_amd.exact import ExactPagedCache
from turboquant_amd.fp8 import Fp8PagedCache
from turboquant_amd.rotary import inverse_frequencies, rotate_heads


_LIBRARY = _ffi.lib()


def real_attend():
    return _LIBRARY.tq_attend


@pytest.fixture
def calls(monkeypatch):
    got, real = [], _LIBRARY

    class Library:
        def __getattr__(self, name):
            return getattr(real, name) if name.endswith("_bytes") else lambda *a: got.append((name, a)) or 0
    monkeypatch.setattr(_ffi, "lib", Library)
    monkeypatch.setattr(_ffi, "native", lambda: None)
    monkeypatch.setattr(_ffi, "require_gpu", lambda t, name: t)
    monkeypatch.setattr(_ffi, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_ffi, "stream_ptr", lambda device: None)
    return got


# ---- rotation in place ------------------------------------------------------------------------------------------------------------

def heads(rows=6, H=4, d=64):
    """Queries and keys of as many heads, and the two as views of one projection."""
    q, k = torch.zeros(rows, H, d), torch.zeros(rows, H, d)
    qkv = torch.zeros(rows, 3 * H * d)
    return (q, k), (qkv[:, : H * d].view(rows, H, d), qkv[:, H * d: 2 * H * d].view(rows, H, d))


def rotate(q, k, out):
    return rotate_heads(q, k, torch.arange(q.shape[0]), inverse_frequencies(q.shape[2]), out=out)


@pytest.mark.parametrize("views", [False, True])
def test_an_output_replaces_its_own_input_only(calls, views):
    """A head is read by the lanes that write it, and by nobody before: true of out=(query, key), not of an output in the other input's place."""
    q, k = heads()[views]
    for out in ((k, q), (k, torch.zeros_like(q)), (torch.zeros_like(q), q), (k, k.clone()), (q.clone(), q)):
        with pytest.raises(ValueError):
            rotate(q, k, out)
    assert not calls
    allowed = (q, k), (q, torch.zeros_like(k)), (torch.zeros_like(q), k)
    for out in allowed:
        assert rotate(q, k, out)[0] is out[0]
    assert [(a[0], a[1], a[19], a[22]) for _, a in calls] == [tuple(t.data_ptr() for t in (q, k, *out)) for out in allowed]


def test_queries_that_are_the_keys(calls):
    """One tensor, or two that share heads: neither may be written."""
    q, new = heads()[0]
    wide = torch.zeros(6, 6, 64)
    for a, b in ((q, q), (wide[:, :4], wide[:, 2:])):
        for out in ((a, new), (new, b), (a, b)):
            with pytest.raises(ValueError):
                rotate(a, b, out)
        assert not calls
        rotate(a, b, (new, new.clone()))
        rotate(a, b, None)
        assert len(calls) == 2
        calls.clear()


def test_outputs_beside_inputs_of_one_projection(calls):
    """Columns that nobody reads may be written."""
    rows, H, d = 6, 4, 64
    x = torch.zeros(rows, 4 * H * d)
    q, k, a, b = (x[:, i * H * d: (i + 1) * H * d].view(rows, H, d) for i in range(4))
    for out in ((a, b), (q, a), (a, k), (q, k)):
        rotate(q, k, out)
    assert len(calls) == 4
    for out in ((a, a), (k, a), (a, q), (x[:, 64: 64 + H * d].view(rows, H, d), k)):
        with pytest.raises(ValueError):
            rotate(q, k, out)
    assert len(calls) == 4


# ---- rows and heads that are alone ------------------------------------------------------------------------------------------------

def cache8(blocks=4, H=2, d=64):
    k = torch.zeros(blocks, 16, H, d, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(blocks, H, dtype=torch.uint8)
    return Fp8PagedCache(k, k.clone(), s, s.clone())


def step(*runs):
    starts = torch.tensor([0, *runs]).cumsum(0).to(torch.int32)
    return starts, torch.arange(4, dtype=torch.int32).expand(len(runs), 4).contiguous(), torch.tensor([max(1, r) for r in runs], dtype=torch.int32)


@pytest.mark.parametrize("shape,strides", [((1, 2, 64), (1001, 64, 1)), ((3, 1, 64), (64, 7, 1)), ((1, 1, 64), (3, 5, 1))])
def test_a_step_between_rows_that_nobody_takes(calls, shape, strides):
    """torch calls a tensor contiguous whatever the stride of a dimension of one element: the library is not given it."""
    x = torch.zeros(2048).as_strided(shape, strides)
    cache = cache8(H=shape[1])
    cache.write(x, x, *step(shape[0]))
    rotate_heads(x, x, torch.arange(shape[0]), inverse_frequencies(64))
    y, z = (torch.zeros(2048).as_strided(shape, strides) for _ in range(2))
    got = rotate_heads(x, x.clone(), torch.arange(shape[0]), inverse_frequencies(64), out=(y, z))
    assert got[0] is y and got[1] is z
    rotate_heads(y, z, torch.arange(shape[0]), inverse_frequencies(64), out=(y, z))
    at = {"tq_fp8_write": (4, 5, 6, 7), "tq_rotate_heads": (7, 8, 9, 10, 20, 21, 23, 24)}
    for name, a in calls:
        assert all(a[i] >= 0 and a[i] % 4 == 0 for i in at[name]), (name, [a[i] for i in at[name]])
    assert len(calls) == 4 and calls[0][1][0] == x.data_ptr() and calls[2][1][0] == x.data_ptr()      # (read where it lies)


# ---- memory that a call writes and what it goes by ----------------------------------------------------------------------------------

def over(t, like):
    """A tensor like `like` in the memory of t."""
    return t.view(-1).view(torch.uint8)[: like.numel() * like.element_size()].view(like.dtype).view(like.shape)


def wide_step(ints=1 << 15):
    """A step of two rows whose starts, table and lengths have memory enough behind them for an output or a workspace."""
    starts, table, lens = (torch.zeros(ints, dtype=torch.int32) for _ in range(3))
    return dict(query_start_loc=starts, block_table=table, seq_lens=lens), (starts[:3], table[:8].view(2, 4), lens[:2])


@pytest.mark.parametrize("what", ["query_start_loc", "block_table", "seq_lens"])
def test_attention_does_not_write_what_it_goes_by(calls, what):
    held, args = wide_step()
    cache, q = cache8(), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    work = cache.workspace(2, 4, 64, B=2)
    for call in (lambda **kw: cache.attention(q, *args, **kw), lambda **kw: cache.decode_attention(q, *args[1:], **kw)):
        if what == "query_start_loc" and call(out=torch.zeros_like(q)) is not None and calls[-1][1][3] is None:
            continue                                          # (a decode step has no starts)
        for kw in (dict(out=over(held[what], q)), dict(workspace=over(held[what], work))):
            n = len(calls)
            with pytest.raises(ValueError):
                call(**kw)
            assert len(calls) == n
        call(out=torch.zeros_like(q), workspace=work)
        assert calls[-1][0] == "tq_attend"


@pytest.mark.parametrize("what", ["query_start_loc", "block_table", "seq_lens"])
def test_read_does_not_write_what_it_goes_by(calls, what):
    held, args = wide_step()
    cache, k = cache8(), torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    for out in ((over(held[what], k), k), (k, over(held[what], k))):
        with pytest.raises(ValueError):
            cache.read(*args, out=out)
    assert not calls
    cache.read(*args, out=(k, k.clone()))
    assert calls[-1][0] == "tq_fp8_read"


@pytest.mark.parametrize("what", [0, 1, 2])
@pytest.mark.parametrize("part", ["key_cache", "value_scales"])
def test_write_does_not_write_what_it_goes_by(calls, what, part):
    cache = cache8()
    starts, table, lens = step(1)
    k = torch.zeros(1, 2, 64)
    args = [starts, table[:, :2].contiguous(), lens]
    args[what] = over(cache.tensors()[part], args[what])
    with pytest.raises(ValueError):
        cache.write(k, k, *args)
    assert not calls


@pytest.mark.parametrize("what", ["block_table", "seq_lens"])
def test_exact_decode_does_not_write_what_it_goes_by(calls, what):
    held, args = wide_step()
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    cache, q = ExactPagedCache(k, k.clone()), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    work = cache.workspace(2, 4, 64)
    for kw in (dict(out=over(held[what], q)), dict(workspace=over(held[what], work))):
        with pytest.raises(ValueError):
            cache.decode_attention(q, *args[1:], **kw)
    assert not calls
    cache.decode_attention(q, *args[1:], out=q, workspace=work)
    assert calls[-1][0] == "tq_exact_decode"


# ---- a step of no sequence ------------------------------------------------------------------------------------------------------------

def test_a_step_of_no_sequence_has_no_table():
    """Its table has no rows, so no memory: the rows are nobody's and become zeros.  (Refusals that come after the table's, so that nothing is launched.)"""
    from tests.test_step_host import attend_args, read_args, write_args
    lib = _ffi.lib()
    none = dict(B=0, table=None, lens=None)
    assert lib.tq_attend(*attend_args(**none, kc=1 << 20 | 8)) == -2 and lib.tq_fp8_read(*read_args(**none, kc=1 << 20 | 8)) == -2
    assert lib.tq_fp8_write(*write_args(**none, kc=1 << 20 | 8)) == -2
    assert lib.tq_attend(*attend_args(**none, rows=0)) == 0 and lib.tq_fp8_read(*read_args(**none, rows=0)) == 0


# ---- workspaces -----------------------------------------------------------------------------------------------------------------------------

MIB = 1 << 20


@pytest.mark.parametrize("call,most", [
    # single tokens of 256 sequences in a wide table: 0.27 GB are four splits of 256 x 32 rows of 128 channels 16 times over
    (dict(cache=3, starts=0, rows=256, B=256, Hq=32, Hkv=32, d=128, max_len=131072), 80), (dict(cache=2, starts=0, rows=256, B=256, Hq=16, Hkv=16, d=256, max_len=131072), 80),
    (dict(cache=3, starts=0, rows=256, B=256, Hq=32, Hkv=8, d=128, max_len=131072), 80), (dict(cache=3, starts=0, rows=256, B=256, Hq=32, Hkv=32, d=128, max_len=1 << 24), 80),
    # more sequences than are shared out anew, of which one may be far longer than the others: 256 MiB
    (dict(cache=3, starts=0, rows=300, B=300, Hq=32, Hkv=32, d=128, max_len=1 << 20), 270), (dict(cache=2, rows=3000, B=1000, Hq=64, Hkv=8, d=256, max_len=1 << 20, max_rows=3), 800),
    # three drafted rows each
    (dict(cache=3, rows=768, B=256, Hq=16, Hkv=16, d=256, max_len=131072, max_rows=3), 160), (dict(cache=2, rows=768, B=256, Hq=64, Hkv=8, d=256, max_len=131072, max_rows=3), 400),
    # prompts: what is shared out anew is bounded whatever the number of rows, and a large part of the output only where that is small
    (dict(cache=3, rows=4096, B=2, Hq=32, Hkv=8, d=128, max_len=8192, max_rows=2048), 80), (dict(cache=2, rows=64 * 2048, B=64, Hq=32, Hkv=8, d=128, max_len=6144, max_rows=2048), 120),
    (dict(cache=2, rows=64 * 2048, B=64, Hq=32, Hkv=8, d=256, max_len=1 << 20, max_rows=2048), 200),
    # nothing to share
    (dict(cache=2, rows=8192, B=1, Hq=32, Hkv=8, d=128, max_len=8192, max_rows=8192), 1), (dict(cache=3, starts=0, rows=256, B=256, Hq=32, Hkv=8, d=128, max_len=300), 1)])
def test_workspaces_are_bounded(call, most):
    """By the rows of the step times their splits, and by what is shared out anew: less than 2 x 1024 workgroups' rows (many rows: 2 x 512 of 128)."""
    a = {**dict(dtype=2, cache=2, starts=1, rows=0, B=0, Hq=0, Hkv=0, d=0, max_len=0, max_rows=1, window=0, sinks=0, n_split=0), **call}
    assert 0 < _ffi.lib().tq_attend_bytes(*a.values()) <= most * MIB, _ffi.lib().tq_attend_bytes(*a.values()) / MIB


def test_a_wider_table_takes_no_more_for_ever():
    """A workspace does not grow with the bound of the lengths once there are workgroups enough."""
    need = lambda B, n: _ffi.lib().tq_attend_bytes(2, 3, 0, B, B, 32, 8, 128, n, 1, 0, 0, 0)
    assert need(64, 1 << 17) == need(64, 1 << 20) and need(300, 1 << 20) == need(300, 1 << 24)


# ---- hooks --------------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("window,hooks,warned", [(8, {}, [0, 1, 2]), (None, {}, []), (8, dict(exact_layers=1), [1, 2]), (8, dict(exact_layers=3), []), (0, {}, []), ((7, 0), {}, [0, 1, 2]),
                                                 ((-1, -1), {}, []), ((-1, 3), {}, [0, 1, 2]), ("half", {}, [0, 1, 2])])
def test_a_window_that_pages_do_not_honour_is_said(monkeypatch, caplog, window, hooks, warned):
    from turboquant_amd.integration import batched, vllm as single
    from turboquant_amd.integration.harness import MinimalRunner
    monkeypatch.setattr(batched, "TurboQuantProd", lambda *a, **k: None)
    monkeypatch.setattr(batched, "PagedKVPool", lambda *a, **k: None)
    r = MinimalRunner(n_layers=3, hidden=32, num_heads=4, num_kv_heads=2, head_dim=64, ffn=32, vocab=10, batch=2, max_seq_len=32, device="cpu")
    for lay in r.layers:
        lay.attn.impl.sliding_window = window
    before = single.get_mode()
    try:
        with caplog.at_level("WARNING"):
            states = batched.install_batched_hooks(r, r.num_blocks, mode="hybrid", **hooks)
    finally:
        single.set_mode(before)
    said = [m.getMessage() for m in caplog.records if "sliding window" in m.getMessage()]
    assert len(said) == bool(warned) and all((name in said[0]) == (i in warned) for i, name in enumerate(states) if warned)


def test_starts_without_memory(calls):
    """A zero tensor of torch's own has an address of nothing, which the library takes for a step of single tokens: refused."""
    none = torch._efficientzerotensor(3, dtype=torch.int32)
    cache, q, k = cache8(), torch.zeros(2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 2, 64)
    _, table, lens = step(1, 1)
    for call in (lambda: cache.attention(q, none, table, lens), lambda: cache.write(k, k, none, table, lens), lambda: cache.read(none, table, lens, rows=2)):
        with pytest.raises(ValueError):
            call()
    assert not calls


@pytest.mark.parametrize("table", [torch.zeros(1, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int64), torch.zeros(2, 0, dtype=torch.int32)])
def test_ingesting_needs_a_table_for_every_sequence(calls, table):
    from turboquant_amd.integration.batched import BatchedLayerState
    state = BatchedLayerState(config=None, quantizer=None, pool=None, fp8=cache8())
    kv, lens = torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16), torch.tensor([20, 30])
    with pytest.raises(ValueError):
        state.ingest_paged_cache(kv, table, lens)
    assert not calls and state.tokens_written == 0
    state.ingest_paged_cache(kv, torch.zeros(3, 4, dtype=torch.int32), lens)
    assert [name for name, _ in calls] == ["tq_fp8_write"] and state.tokens_written == 50


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 2.0 ** 127, -1e300])
def test_a_factor_that_is_no_number_is_refused(calls, scale):
    """Masked scores are -inf: times NaN or times infinity less infinity rows that see nothing would not be zeros."""
    from tests.test_step_host import attend_args
    assert real_attend()(*attend_args(scale=scale if abs(scale) < 1e39 else float("inf"))) == -1
    cache, q = cache8(), torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    starts, table, lens = step(1, 1)
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: cache.attention(q, starts, table, lens, scale=scale), lambda: cache.decode_attention(q, table, lens, scale=scale),
                 lambda: ExactPagedCache(k, k.clone()).decode_attention(q, table, lens, scale=scale, window=4)):
        with pytest.raises(ValueError, match="scale"):
            call()
    assert not calls
    cache.attention(q, starts, table, lens, scale=2.0 ** 126)
    assert len(calls) == 1


@pytest.mark.parametrize("planned", [16400, 32784, 100000, 1 << 20])
def test_a_workspace_serves_narrower_tables(calls, planned):
    """A workspace for up to so many tokens is enough for steps of that bound, however wide the table is that they come with."""
    q = torch.zeros(1, 16, 256, dtype=torch.bfloat16)
    cache = cache8(H=2, d=256)
    work, rows = cache.workspace(1, 16, planned), cache.workspace(1, 16, planned, B=1)
    for pages in (1, 64, 1000, 1024, 2048, planned // 16 + 1):
        table, lens, starts = torch.zeros(1, pages, dtype=torch.int32), torch.tensor([10], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
        cache.decode_attention(q, table, lens, workspace=work, max_len=planned)
        cache.attention(q, starts, table, lens, workspace=rows, max_len=planned)
    assert len(calls) == 12


def test_more_workgroups_than_a_launch_has():
    """A launch has less than 2^32 threads, 2^24 workgroups of 256: what takes more is refused in front of it."""
    from tests.test_step_host import read_args, rotate_args, write_args
    lib = _LIBRARY
    assert lib.tq_rotate_heads(*rotate_args(rows=1 << 26)) == -1
    assert lib.tq_fp8_write(*write_args(rows=1 << 28)) == -1 and lib.tq_fp8_read(*read_args(rows=1 << 28)) == -1
    need = lambda rows, **kw: lib.tq_attend_bytes(*{**dict(dtype=2, cache=2, starts=1, rows=rows, B=4, Hq=32, Hkv=8, d=256, max_len=1 << 16, max_rows=rows, window=0, sinks=0, n_split=0), **kw}.values())
    assert need(1 << 20) > 0 and need(1 << 17, n_split=128) == 0 and need(1 << 17, n_split=64) > 0                 # (the join of over 64 splits: a workgroup for 64 channels of a row)
    assert need(1 << 24, Hkv=32, max_rows=1 << 24) == 0 and need(1 << 22, B=1 << 22, Hq=8, d=64, max_rows=1, max_len=16) == 0
