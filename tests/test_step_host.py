"""What the entry points of a step refuse before they launch anything, their plans, and what the Python calls refuse: no GPU is touched."""

import math

import pytest
import torch

from turboquant_amd import _ffi
from turboquant_amd.attend import overlaps, plan_bytes, seen_by, step_starts
from turboquant_amd.exact import ExactPagedCache
from turboquant_amd.fp8 import Fp8PagedCache
from turboquant_amd.integration.batched import _window_of, install_batched_hooks
from turboquant_amd.integration.harness import DenseBackend, MinimalRunner
from turboquant_amd.rotary import inverse_frequencies, rotate_heads

P = 1 << 20                                  # an aligned address that no refused call looks at
BIG = 1 << 31


def arguments(given, kw):
    assert set(kw) <= set(given)
    return list({**given, **kw}.values())


def write_args(**kw):
    return arguments(dict(k=P, v=P, dtype=2, rows=16, ks_t=256, ks_h=128, vs_t=256, vs_h=128, starts=P, B=2, Hkv=2, d=128, kc=P, vc=P, ksc=P, vsc=P,
                          cs_blk=16 * 256, cs_t=256, cs_h=128, num_blocks=4, table=P, bt_stride=2, lens=P, stream=None), kw)


CACHE = [(dict(kc=None), -3), (dict(vc=None), -3), (dict(ksc=None), -3), (dict(vsc=None), -3), (dict(table=None), -3), (dict(lens=None), -3), (dict(starts=None), -3),
         (dict(Hkv=0), -1), (dict(d=0), -1), (dict(d=96), -2), (dict(d=320), -2), (dict(num_blocks=0), -1), (dict(bt_stride=0), -1), (dict(bt_stride=-BIG), -1),
         (dict(B=-1), -1), (dict(rows=-1), -1), (dict(rows=BIG), -1), (dict(cs_t=-16), -2), (dict(cs_t=(1 << 24) + 16), -2), (dict(cs_blk=8), -2),
         (dict(cs_h=100), -2), (dict(kc=P + 8), -2), (dict(vc=P + 1), -2), (dict(dtype=3), -1), (dict(dtype=-1), -1)]


@pytest.mark.parametrize("bad,rc", CACHE + [
    (dict(k=None), -3), (dict(v=None), -3), (dict(ks_t=-8), -1), (dict(vs_h=-8), -1), (dict(ks_t=4), -2), (dict(vs_t=258), -2), (dict(dtype=0, ks_h=130), -2),
    (dict(k=P + 8), -2), (dict(v=P + 4), -2), (dict(bt_stride=-2), -1)])
def test_write_refuses(bad, rc):
    assert _ffi.lib().tq_fp8_write(*write_args(**bad)) == rc


def read_args(**kw):
    return arguments(dict(k=P, v=P, dtype=2, rows=16, starts=P, B=2, Hkv=2, d=128, kc=P, vc=P, ksc=P, vsc=P, cs_blk=16 * 256, cs_t=256, cs_h=128,
                          num_blocks=4, table=P, bt_stride=2, lens=P, fill=1, stream=None), kw)


@pytest.mark.parametrize("bad,rc", CACHE + [(dict(k=None), -3), (dict(v=None), -3), (dict(k=P + 8), -2), (dict(v=P + 2), -2)])
def test_read_refuses(bad, rc):
    assert _ffi.lib().tq_fp8_read(*read_args(**bad)) == rc


def attend_args(**kw):
    return arguments(dict(q=P, dtype=2, rows=16, starts=P, B=2, Hq=8, Hkv=2, d=128, cache=3, kc=P, vc=P, ksc=P, vsc=P, cs_blk=16 * 256, cs_t=256, cs_h=128,
                          num_blocks=4, table=P, bt_stride=2, lens=P, scale=0.1, max_len=32, max_rows=16, window=0, sinks=0, out=P, fill=1, workspace=P,
                          n_split=0, stream=None), kw)


@pytest.mark.parametrize("bad,rc", [(dict(kc=None), -3), (dict(vc=None), -3), (dict(ksc=None), -3), (dict(vsc=None), -3), (dict(table=None), -3), (dict(lens=None), -3),
    (dict(q=None), -3), (dict(out=None), -3), (dict(workspace=None), -3), (dict(dtype=0), -1), (dict(dtype=3), -1), (dict(cache=0), -1), (dict(cache=1), -1),
    (dict(rows=-1), -1), (dict(rows=BIG), -1), (dict(B=-1), -1), (dict(Hq=0), -1), (dict(Hkv=0), -1), (dict(Hq=9), -1), (dict(d=96), -1), (dict(d=320), -1),
    (dict(Hq=2050, Hkv=2), -1), (dict(max_len=-1), -1), (dict(max_len=BIG), -1), (dict(max_rows=-1), -1), (dict(window=-1), -1), (dict(sinks=-1), -1),
    (dict(n_split=-1), -1), (dict(n_split=1025), -1), (dict(starts=None, rows=3), -1), (dict(num_blocks=0), -1), (dict(bt_stride=0), -1), (dict(cs_t=8), -2),
    (dict(cs_blk=-16), -2), (dict(kc=P + 8), -2), (dict(cache=2, cs_h=132), -2), (dict(cache=2, vc=P + 2), -2), (dict(q=P + 8), -2), (dict(out=P + 4), -2),
    (dict(workspace=P + 8), -1)])
def test_attention_refuses(bad, rc):
    assert _ffi.lib().tq_attend(*attend_args(**bad)) == rc


def rotate_args(**kw):
    return arguments(dict(q=P, k=P, dtype=2, rows=16, Hq=8, Hkv=2, d=128, qs_t=1280, qs_h=128, ks_t=1280, ks_h=128, pos=P, wide=0, inv=P, rotary=128,
                          interleaved=0, qw=P, kw=P, eps=1e-6, qo=P, qo_t=1024, qo_h=128, ko=P, ko_t=256, ko_h=128, stream=None), kw)


@pytest.mark.parametrize("bad,rc", [(dict(q=None), -3), (dict(k=None), -3), (dict(qo=None), -3), (dict(ko=None), -3), (dict(pos=None), -3), (dict(inv=None), -3),
    (dict(dtype=3), -1), (dict(rows=-1), -1), (dict(rows=BIG), -1), (dict(Hq=-1), -1), (dict(Hq=0, Hkv=0), -1), (dict(Hq=1 << 24), -1), (dict(d=0), -1),
    (dict(rotary=-8), -1), (dict(rotary=136), -1), (dict(rotary=12), -2), (dict(d=100, rotary=64), -2), (dict(d=520), -2), (dict(qs_t=-4), -2), (dict(ko_h=130), -2),
    (dict(q=P + 4), -2), (dict(kw=P + 2), -2), (dict(dtype=0, k=P + 8), -2)])
def test_rotation_refuses(bad, rc):
    assert _ffi.lib().tq_rotate_heads(*rotate_args(**bad)) == rc


def test_nothing_to_do_launches_nothing():
    lib = _ffi.lib()
    assert lib.tq_fp8_write(*write_args(rows=0)) == 0 and lib.tq_fp8_read(*read_args(rows=0)) == 0
    assert lib.tq_attend(*attend_args(rows=0, workspace=None)) == 0 and lib.tq_attend(*attend_args(rows=0, B=0, starts=None, workspace=None, lens=None)) == 0
    assert lib.tq_rotate_heads(*rotate_args(rows=0)) == 0


def test_plans():
    need = _ffi.lib().tq_attend_bytes
    #            dtype cache starts rows B Hq Hkv d max_len max_rows window sinks n_split
    assert need(2, 3, 1, 16, 2, 9, 2, 128, 32, 16, 0, 0, 0) == 0 and need(2, 1, 1, 16, 2, 8, 2, 128, 32, 16, 0, 0, 0) == 0
    assert need(2, 3, 0, 16, 2, 8, 2, 128, 32, 16, 0, 0, 0) == 0                             # (one row per sequence)
    assert need(2, 3, 1, BIG - 1, 2, 1024, 1, 256, 1 << 20, 4096, 0, 0, 1024) == 0           # (more workgroups than a grid holds)
    one = need(2, 3, 1, 16, 2, 8, 2, 128, 32, 16, 0, 0, 1)
    assert one > 0 and need(2, 3, 1, 16, 2, 8, 2, 128, 32, 16, 0, 0, 0) > 0
    # a window of few tokens takes fewer splits of a long cache than none does
    assert need(2, 3, 0, 1, 1, 8, 2, 128, 1 << 20, 1, 256, 4, 0) < need(2, 3, 0, 1, 1, 8, 2, 128, 1 << 20, 1, 0, 0, 0)


def test_windows():
    assert seen_by(None, 0) == (0, 0) and seen_by(5, 2) == (5, 2) and seen_by(BIG - 1, 0) == (BIG - 1, 0)
    for window, sinks in ((None, 1), (0, 0), (-1, 0), (BIG, 0), (4, -1), (4, BIG)):
        with pytest.raises(ValueError):
            seen_by(window, sinks)


class Impl:
    def __init__(self, **kw):
        self.__dict__.update(kw)


@pytest.mark.parametrize("named,want", [({}, (None, 0)), (dict(sliding_window=None, sink_tokens=4), (None, 0)), (dict(sliding_window=64), (64, 0)),
    (dict(sliding_window=64, sink_tokens=4), (64, 4)), (dict(sliding_window=(63, 0)), (64, 0)), (dict(sliding_window=(-1, -1)), (None, 0)),
    (dict(sliding_window=0), (None, 0)), (dict(sliding_window=[0, 0], sink_tokens=1), (1, 1))])
def test_windows_of_backends(named, want):
    assert _window_of("layer", Impl(**named)) == want


@pytest.mark.parametrize("named", [dict(sliding_window=(8, 1)), dict(sliding_window=8, sink_tokens=-1), dict(sliding_window=BIG)])
def test_windows_of_backends_that_are_refused(named):
    with pytest.raises(ValueError):
        _window_of("layer", Impl(**named))


def test_tensors_on_the_host_are_refused():
    k = torch.zeros(4, 16, 2, 64)
    scales = torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises(RuntimeError):
        Fp8PagedCache(k.to(torch.float8_e4m3fn), k.to(torch.float8_e4m3fn), scales, scales.clone())
    with pytest.raises(RuntimeError):
        Fp8PagedCache.allocate(4, 2, 64, "cpu")
    with pytest.raises(RuntimeError):
        rotate_heads(k[0], k[0], torch.arange(16), inverse_frequencies(64))
    with pytest.raises(RuntimeError):
        ExactPagedCache(k.bfloat16(), k.bfloat16())


def test_starts():
    with pytest.raises(ValueError):
        step_starts(torch.device("cpu"), torch.zeros(0, dtype=torch.int32))
    with pytest.raises(ValueError):
        step_starts(torch.device("cpu"), torch.zeros(2, 2, dtype=torch.int32))
    t, B = step_starts(torch.device("cpu"), torch.tensor([0, 9, 3, 9, 7])[::2])
    assert B == 2 and t.tolist() == [0, 3, 7] and t.dtype == torch.int32


def test_overlaps():
    t = torch.zeros(8, 4)
    assert overlaps(t, t[7]) and not overlaps(t[:4], t[4:]) and not overlaps(t[:0], t) and overlaps(t[::2], t[1::2])


def test_inverse_frequencies():
    got = inverse_frequencies(8, 10000.0)
    assert got.dtype == torch.float64 and torch.allclose(got, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)


SIZE = dict(n_layers=2, hidden=32, num_heads=4, num_kv_heads=2, ffn=32, vocab=10, batch=2, max_seq_len=32)


@pytest.mark.parametrize("head_dim,hooks,says", [(64, dict(fp8_layers=1), "GPU"), (64, dict(exact_layers=-1), "negative"), (64, dict(fp8_layers=-1), "negative"),
                                                 (320, dict(exact_layers=1), "320"), (64, dict(exact_layers=1, no_alloc=True), "no_alloc")])
def test_hooks_refuse_before_they_touch_a_layer(head_dim, hooks, says):
    from turboquant_amd.integration import vllm as single
    r = MinimalRunner(device="cpu", head_dim=head_dim, sliding_window=8, **SIZE)
    before = single.get_mode()
    with pytest.raises(ValueError, match=says):
        install_batched_hooks(r, r.num_blocks, mode="full_tq", **hooks)
    assert single.get_mode() == before and not hasattr(r, "_tq_layer_states") and all("forward" not in vars(lay.attn.impl) for lay in r.layers)


def test_the_backends_window():
    """DenseBackend against the definition, on the host."""
    H, G, d, n, window, sinks = 2, 2, 16, 40, 7, 3
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, H, d, generator=g) for _ in range(2))
    q = torch.randn(5, H * G, d, generator=g)
    impl = DenseBackend(H * G, H, d, window, sinks)
    cache = torch.zeros(2, 3, 16, H, d)
    impl.do_kv_cache_update(None, k, v, cache, torch.arange(n))
    meta = Impl(num_actual_tokens=5, seq_lens_cpu=torch.tensor([n]), query_start_loc_cpu=torch.tensor([0, 5]), block_table=torch.tensor([[0, 1, 2]]))
    got = impl.forward(None, q, None, None, cache, meta)
    for i in range(5):
        p = n - 5 + i
        t = torch.tensor([t for t in range(p + 1) if t > p - window or t < sinks])
        s = torch.einsum("hd,nhd->hn", q[i].double(), k[t].double().repeat_interleave(G, 1)) / math.sqrt(d)
        want = torch.einsum("hn,nhd->hd", s.softmax(-1), v[t].double().repeat_interleave(G, 1))
        # sums of 40 products in 32 bits, of numbers below 5
        assert (got[i].double() - want).abs().max() <= 40 * 5 * 2.0 ** -23


def test_plan_bytes_refuses():
    class Cache:
        _tag, num_kv_heads, head_dim = _ffi.TQ_E4M3, 2, 128
    for bad in (dict(n_split=-1), dict(max_len=-1), dict(max_rows=-1), dict(n_split=1025), dict(Hq=9)):
        kw = dict(rows=4, B=2, Hq=8, max_len=100, max_rows=2, window=0, sinks=0, n_split=0)
        with pytest.raises(ValueError):
            plan_bytes(Cache, torch.bfloat16, True, **{**kw, **bad})
