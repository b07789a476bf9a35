"""Operators over 4-bit caches, eviction and beams: every refusal of an argument comes before a device is needed; format of the cache."""
import ctypes as C

import numpy as np
import pytest

import plain_cache4 as P
from conftest import load_package

lcu = load_package()
A = 1 << 20  # an address that nothing reads: the calls below are refused


def refused(rc, words):
    assert rc == 2 and words.encode() in lcu.lib.lcu_last_error(), (rc, lcu.lib.lcu_last_error())


def append(**k):
    a = dict(kc=A, ks=A, vc=A, vs=A, qo=A, q=A, ldq=512, k=A, v=A, ldkv=256, lengths=A, positions=None, seqs=1, m=1, heads=4, kv=2, hd=128, bs=32, ctx=64,
             theta=10000.0, dtype=0, stream=None)
    return lcu.lib.lcu_cache4_append(*{**a, **k}.values())


@pytest.mark.parametrize("change,words", [
    (dict(kc=None), "null pointer"), (dict(vs=None), "null pointer"), (dict(k=None), "null pointer"), (dict(lengths=None), "null pointer"), (dict(qo=None), "null pointer"),
    (dict(hd=96), "head_dim 96"), (dict(hd=64, bs=128), "block size 128"), (dict(bs=16), "block size 16"), (dict(bs=0), "block size 0"), (dict(seqs=0), "no sequences"),
    (dict(kv=0), "no sequences"), (dict(ctx=0), "no sequences"), (dict(kc=A + 8), "16-byte aligned"), (dict(ks=A + 2), "16-byte aligned"), (dict(dtype=2), "number format 2"),
    (dict(m=0), "no rows"), (dict(heads=0), "no rows"), (dict(ldkv=248), "row strides"), (dict(ldq=516), "row strides"), (dict(k=A + 4), "16-byte aligned"),
    (dict(ldq=520, qo=A), "must be dense"), (dict(lengths=A + 2), "4-byte aligned"), (dict(positions=A + 1), "4-byte aligned"), (dict(theta=-1.0), "theta"), (dict(theta=float("nan")), "theta"), (dict(seqs=1 << 16, m=1 << 16), "too many")])
def test_append_refuses(change, words):
    refused(append(**change), words)


def attend(**k):
    a = dict(out=A, ldo=512, w=None, beta=0.0, q=A, ldq=512, kc=A, ks=A, vc=A, vs=A, lengths=A, seqs=1, m=1, heads=4, kv=2, hd=128, bs=32, ctx=64, most=64, dtype=0,
             ws=A, bytes=1 << 40, stream=None)
    return lcu.lib.lcu_attention_cache4(*{**a, **k}.values())


@pytest.mark.parametrize("change,words", [
    (dict(out=None), "null pointer"), (dict(q=None), "null pointer"), (dict(lengths=None), "null pointer"), (dict(kc=None), "null pointer"), (dict(heads=3), "3 heads over 2"),
    (dict(m=0), "0 rows"), (dict(most=65), "exceed the cache"), (dict(most=0), "exceed the cache"), (dict(ldo=504), "row strides"), (dict(ldq=500), "row strides"),
    (dict(q=A + 8), "16-byte aligned"), (dict(out=A + 2), "16-byte aligned"), (dict(dtype=2), "number format 2"), (dict(hd=80), "head_dim 80"),
    (dict(m=200, ws=None), "workspace"), (dict(lengths=A + 1), "4-byte aligned"), (dict(w=A + 2), "4-byte aligned"), (dict(w=A, ws=None), "workspace"), (dict(w=A, bytes=0), "workspace"), (dict(w=A, ws=A + 4), "workspace"), (dict(seqs=40000), "too many")])
def test_attention_refuses(change, words):
    refused(attend(**change), words)


def test_read_refuses():
    def read(**k):
        a = dict(ko=A, vo=A, kc=A, ks=A, vc=A, vs=A, first=None, seqs=1, count=1, kv=2, hd=128, bs=32, ctx=64, dtype=0, stream=None)
        return lcu.lib.lcu_cache4_read(*{**a, **k}.values())

    refused(read(ko=None, vo=None), "nothing to read")
    refused(read(count=0), "nothing to read")
    refused(read(ko=A + 4), "16-byte aligned")
    refused(read(dtype=5), "number format 5")
    refused(read(bs=24), "block size 24")
    refused(read(first=A + 2), "4-byte aligned")


def planes(*addresses):
    return (C.c_void_p * len(addresses))(*addresses)


def test_evict_refuses():
    def evict(**k):
        a = dict(dst=planes(A), src=planes(A), rb=(C.c_int * 1)(64), n=1, w=A, kept=A, lo=None, lengths=A, seqs=1, kv=2, ctx=64, dctx=64, keep=10, recent=2, stream=None)
        return lcu.lib.lcu_cache_evict(*{**a, **k}.values())

    refused(evict(n=9), "9 planes")
    refused(evict(n=-1), "-1 planes")
    refused(evict(src=planes(None)), "plane 0 is a null pointer")
    refused(evict(rb=(C.c_int * 1)(3)), "rows of 3 bytes")
    refused(evict(rb=(C.c_int * 1)(0)), "rows of 0 bytes")
    refused(evict(dst=planes(A + 1)), "odd address")
    refused(evict(w=None), "null pointer")
    refused(evict(kept=None), "null pointer")
    refused(evict(keep=0), "keep 0 rows")
    refused(evict(keep=65), "keep 65 rows")
    refused(evict(recent=11), "keep 10 rows")
    refused(evict(recent=-1), "keep 10 rows")
    refused(evict(dst=planes(1 << 24), dctx=9), "into 9")
    refused(evict(dctx=32), "in place")
    refused(evict(seqs=0), "0 sequences")
    refused(evict(w=A + 2), "4-byte aligned")
    refused(evict(lo=A + 1), "4-byte aligned")


def test_reorder_refuses():
    def reorder(**k):
        a = dict(dst=planes(A), src=planes(A), rb=(C.c_int * 1)(64), n=1, parents=A, lengths=A, groups=1, beams=4, kv=2, ctx=64, stream=None)
        return lcu.lib.lcu_cache_reorder(*{**a, **k}.values())

    refused(reorder(n=0), "0 planes")
    refused(reorder(parents=None), "null pointer")
    refused(reorder(beams=0), "0 beams")
    refused(reorder(beams=33), "33 beams")
    refused(reorder(groups=0), "0 groups")
    refused(reorder(ctx=0), "0 rows")
    refused(reorder(parents=A + 2), "4-byte aligned")


def test_beam_select_refuses():
    def select(**k):
        a = dict(parents=A, tokens=A, out=A, logits=A, ld=100, dtype=0, scores=A, groups=1, beams=4, vocab=100, n=4, ws=A, bytes=1 << 40, stream=None)
        return lcu.lib.lcu_beam_select(*{**a, **k}.values())

    refused(select(logits=None), "null pointer")
    refused(select(scores=None), "null pointer")
    refused(select(dtype=3), "number format 3")
    refused(select(beams=33), "33 beams")
    refused(select(ld=99), "vocabulary of 100 in rows of 99")
    refused(select(vocab=0), "vocabulary of 0")
    refused(select(n=0), "0 continuations")
    refused(select(n=65), "65 continuations")
    refused(select(beams=1, vocab=3, ld=3, n=4), "4 continuations")
    refused(select(logits=A + 1), "aligned to their type")
    refused(select(dtype=2, logits=A + 2), "aligned to their type")
    refused(select(bytes=16), "workspace")
    refused(select(ws=None), "workspace")
    refused(select(tokens=A + 2), "4-byte aligned")


def test_workspaces_of_senseless_sizes():
    """Queries of sizes that a call would refuse return 0; sensible ones grow with the rows."""
    w = lcu.lib.lcu_attention_cache4_workspace
    assert w(0, 1, 4, 2, 128, 64, 1) == 0 and w(1, 0, 4, 2, 128, 64, 1) == 0 and w(1, 1, 1, 2, 128, 64, 0) == 0 and w(1, 1, 4, 0, 128, 64, 0) == 0
    assert w(1, 1, 4, 2, 128, 0, 0) == 0 and w(1, -5, 4, 2, 128, 64, 0) == 0
    assert 0 < w(1, 500, 4, 2, 128, 600, 0) < w(1, 500, 4, 2, 128, 6000, 0)
    assert w(1, 1, 32, 32, 128, 40000, 1) >= 32 * 40000 * 4 + w(1, 1, 32, 32, 128, 40000, 0)
    b = lcu.lib.lcu_beam_select_workspace
    assert b(0, 1, 5, 1) == 0 and b(1, 1, -5, 1) == 0 and b(2, 4, 32000, 4) > 0


def test_valid_calls_need_a_device():
    if lcu.lib.lcu_device_count() > 0:
        pytest.skip("a GPU is present")
    for call in (append, attend):
        assert call() == 1 and b"no CUDA device" in lcu.lib.lcu_last_error()
    with pytest.raises(lcu.LcuError, match="no CUDA device"):
        lcu.beam_select(np.zeros((1, 2, 10), np.float32), np.zeros((1, 2), np.float32), 2)


@pytest.mark.parametrize("hd,bs", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
def test_values_of_the_cache_are_exact_halves(hd, bs):
    """Seven-bit scales: every value (code - 7.5) * scale is a half; rows come back within half a step (the largest magnitude of a block may
    lie up to 2^-7 of itself, 0.06 steps, above 7.5 scales: still nearest to the last code)."""
    rng = np.random.default_rng(hd + bs)
    x = (rng.standard_normal((400, hd)) * 10.0 ** rng.uniform(-2, 3, (400, 1))).astype(np.float32)
    s = P.scales_of(x, bs)
    c = P.codes_of(x, s, bs)
    v = P.values_of(c, s, bs)
    assert (P.unpack(P.pack(c)) == c).all()
    assert (v.astype(np.float16).astype(np.float64) == v).all()
    assert (np.abs(v - x) <= 0.5 * np.repeat(s.astype(np.float64), bs, -1) * (1 + 2.0 ** -7) + 2.0 ** -7 * np.abs(x)).all()


def test_plain_eviction_and_beams():
    w = np.array([5, 1, np.nan, 1, 9, 0, 2], np.float32)
    assert P.evict(w, 7, 4, 2) == [0, 4, 5, 6]
    assert P.evict(w, 6, 4, 0) == [0, 1, 3, 4] and P.evict(w, 6, 5, 0) == [0, 1, 3, 4, 5]
    assert P.evict(w, 3, 4, 1) == [0, 1, 2] and P.evict(w, -1, 4, 1) == []
    p, t, s = P.beam_select(np.array([[0.0, 1.0], [0.0, 1.0]]), np.array([-1.0, -1.0]), 4)
    assert p.tolist() == [0, 1, 0, 1] and t.tolist() == [1, 1, 0, 0]


def cache_without_planes(**k):
    """As Cache4 makes it, without a device: the calls below are refused before anything is allocated."""
    c = object.__new__(lcu.Cache4)
    a = dict(n_seqs=4, n_kv=2, hd=64, ctx=32, bs=32, dtype=0, lengths=np.zeros(4, np.int32), positions=np.zeros(4, np.int32), planes=[], row_bytes=[])
    c.__dict__.update({**a, **k})
    return c


def rows(seqs, m, width):
    return np.zeros((seqs, m, width), np.uint16)


@pytest.mark.parametrize("call", [
    lambda c: c.append(rows(3, 2, 256), rows(4, 2, 128), rows(4, 2, 128)),   # fewer sequences than the cache has
    lambda c: c.append(rows(4, 2, 256), rows(4, 1, 128), rows(4, 2, 128)),   # fewer keys than queries
    lambda c: c.append(rows(4, 2, 256), rows(4, 2, 128), rows(4, 1, 128)),
    lambda c: c.append(rows(4, 2, 256), rows(4, 2, 128), rows(4, 2, 64)),    # values of one head
    lambda c: c.append(rows(4, 2, 200), rows(4, 2, 128), rows(4, 2, 128)),   # heads cut off
    lambda c: c.append(rows(4, 0, 256), rows(4, 0, 128), rows(4, 0, 128)),
    lambda c: c.attend(rows(1, 2, 256)),
    lambda c: c.attend(rows(4, 2, 100)),
    lambda c: c.attend(np.zeros((4, 256), np.uint16)),
    lambda c: c.evict(0, 0),
    lambda c: c.evict(33, 0),
    lambda c: c.reorder(np.zeros((1, 2), np.int32)),                         # two beams of four sequences
    lambda c: c.reorder(np.zeros((2, 4), np.int32)),                         # eight
    lambda c: c.reorder(np.zeros(4, np.int32)),
    lambda c: c.read(0),
    lambda c: c.read(2, first=[0, 0])])
def test_cache_refuses_arrays_of_other_shapes(call):
    with pytest.raises(lcu.LcuError, match="Cache4"):
        call(cache_without_planes())


@pytest.mark.parametrize("lengths", [np.zeros(3, np.int32), np.zeros(4), np.zeros((4, 1), np.int32)])
def test_cache_refuses_lengths_of_other_shapes(lengths):
    c = cache_without_planes(lengths=lengths)
    for call in (lambda: c.append(rows(4, 1, 256), rows(4, 1, 128), rows(4, 1, 128)), lambda: c.attend(rows(4, 1, 256)), lambda: c.evict(8, 0),
                 lambda: c.reorder(np.zeros((1, 4), np.int32))):
        with pytest.raises(lcu.LcuError, match="Cache4"):
            call()


@pytest.mark.parametrize("change", [dict(n_seqs=0), dict(n_kv_heads=0), dict(ctx_len=0), dict(head_dim=96), dict(bs=16), dict(head_dim=64, bs=128), dict(dtype="float32")])
def test_cache_of_senseless_sizes(change):
    with pytest.raises(lcu.LcuError, match="Cache4"):
        lcu.Cache4(**{**dict(n_seqs=1, n_kv_heads=1, head_dim=128, ctx_len=8), **change})


@pytest.mark.parametrize("logits,scores,n_out,dtype", [
    (np.zeros((1, 2, 8), np.uint16), np.zeros((1, 2)), 2, "float32"),    # half as many bytes as the format says
    (np.zeros((1, 2, 8)), np.zeros((1, 2)), 2, "float32"),
    (np.zeros((1, 2, 8), np.float32), np.zeros((1, 2)), 2, "bfloat16"),
    (np.zeros((1, 2, 8), np.float32), np.zeros((1, 2)), 2, "float64"),
    (np.zeros((1, 2, 8), np.float32), np.zeros((1, 1)), 2, "float32"),
    (np.zeros((2, 8), np.float32), np.zeros(2), 2, "float32"),
    (np.zeros((0, 2, 8), np.float32), np.zeros((0, 2)), 2, "float32"),
    (np.zeros((1, 2, 8), np.float32), np.zeros((1, 2)), 0, "float32")])
def test_beam_selection_refuses_arrays_of_other_shapes(logits, scores, n_out, dtype):
    with pytest.raises(lcu.LcuError, match="beam_select"):
        lcu.beam_select(logits, scores, n_out, dtype)


@pytest.mark.parametrize("call", [
    lambda c: c.append(rows(4, 1, 256).view(np.float16), rows(4, 1, 128), rows(4, 1, 128)),  # numbers, which would be cut to whole ones
    lambda c: c.append(rows(4, 1, 256), rows(4, 1, 128).astype(np.float32), rows(4, 1, 128)),
    lambda c: c.append(rows(4, 1, 256), rows(4, 1, 128), rows(4, 1, 128).astype(np.float64)),
    lambda c: c.attend(np.full((4, 1, 256), 0.7, np.float16)),
    lambda c: c.reorder(np.full((1, 4), 0.9)),
    lambda c: c.reorder(np.full((1, 4), 2 ** 32)),                                           # would be beam 0
    lambda c: c.read(1, first=np.full(4, 2 ** 32 + 1))])
def test_cache_refuses_numbers_that_are_no_bit_patterns_or_whole_ones(call):
    with pytest.raises(lcu.LcuError, match="Cache4: .*(patterns|do not hold)"):
        call(cache_without_planes())


@pytest.mark.parametrize("change", [dict(lengths=np.full(4, 2 ** 32)), dict(positions=np.full(4, -2 ** 31 - 1))])
def test_cache_refuses_lengths_beyond_32_bits(change):
    with pytest.raises(lcu.LcuError, match="Cache4: .*do not hold"):
        cache_without_planes(**change).append(rows(4, 1, 256), rows(4, 1, 128), rows(4, 1, 128))


HEAD = 64 * 64  # bytes of a head's 64 rows of 64


@pytest.mark.parametrize("dst,src,rb,dctx,words", [
    ([0, 0], [0, 0], [64, 64], 64, "destinations of planes 0 and 1"),                            # the same plane twice
    ([8 * HEAD, 8 * HEAD], [0, 2 * HEAD], [64, 64], 64, "destinations of planes 0 and 1"),
    ([8 * HEAD, 9 * HEAD - 64], [0, 2 * HEAD], [32, 64], 64, "destinations of planes 0 and 1"),  # the last row of one
    ([HEAD], [0], [64], 64, "plane 0 overlaps the source of plane 0"),                           # moved on by a head
    ([2 * HEAD - 64], [0], [64], 16, "plane 0 overlaps the source of plane 0"),
    ([8 * HEAD, 2 * HEAD], [0, 2 * HEAD + 64], [64, 64], 64, "plane 1 overlaps the source of plane 1"),
    ([2 * HEAD, 8 * HEAD], [0, 2 * HEAD], [64, 64], 64, "plane 0 overlaps the source of plane 1"),
    ([2 * HEAD, 2 * HEAD], [0, 2 * HEAD], [64, 64], 64, "plane 0 overlaps the source of plane 1")])  # which is moved in place
def test_planes_that_overlap_are_refused(dst, src, rb, dctx, words):
    d, s = planes(*[A + x for x in dst]), planes(*[A + x for x in src])
    n = len(dst)
    refused(lcu.lib.lcu_cache_evict(d, s, (C.c_int * n)(*rb), n, A, A, None, A, 1, 2, 64, dctx, 10, 2, None), words)
    if dctx == 64:
        refused(lcu.lib.lcu_cache_reorder(d, s, (C.c_int * n)(*rb), n, A, A, 1, 2, 1, 64, None), words)


def test_planes_side_by_side_are_taken():
    """Neighbours that touch, and a plane that goes to another place and is moved in place as well."""
    if lcu.lib.lcu_device_count() > 0:
        pytest.skip("a GPU is present: these addresses are none")
    d, s, rb = planes(A, A + 2 * HEAD, A + 4 * HEAD), planes(A, A + 6 * HEAD, A), (C.c_int * 3)(64, 64, 64)
    assert lcu.lib.lcu_cache_evict(d, s, rb, 3, A, A, None, A, 1, 2, 64, 64, 10, 2, None) == 1 and b"no CUDA device" in lcu.lib.lcu_last_error()
    assert lcu.lib.lcu_cache_reorder(d, s, rb, 3, A, A, 1, 2, 1, 64, None) == 1 and b"no CUDA device" in lcu.lib.lcu_last_error()
    assert lcu.lib.lcu_cache_evict(d, s, rb, 2, A, A, None, A, 1 << 10, 1 << 9, 1 << 25, 1 << 25, 10, 2, None) == 2  # (planes of 2^50 bytes do overlap)


@pytest.mark.parametrize("change", [dict(heads=5), dict(hd=96), dict(most=2 ** 31 - 1), dict(most=1 << 26), dict(m=2 ** 31 - 1), dict(m=1 << 26), dict(seqs=2 ** 31 - 1),
                                    dict(seqs=1 << 15), dict(seqs=1 << 30, m=1 << 25, heads=1 << 9), dict(heads=1 << 18), dict(m=1 << 25, heads=64),
                                    dict(seqs=16384, m=32, most=(1 << 26) - 1), dict(seqs=16384, m=2000, heads=2, most=(1 << 26) - 1)])
def test_workspaces_of_sizes_that_are_refused(change):
    """0, whatever the numbers' products, and the call says so."""
    a = {**dict(seqs=1, m=500, heads=4, kv=2, hd=128, most=100), **change}
    for weights in (0, 1):
        assert lcu.lib.lcu_attention_cache4_workspace(a["seqs"], a["m"], a["heads"], a["kv"], a["hd"], a["most"], weights) == 0
    a = {**a, "ctx": a["most"], "ldq": 1 << 26, "ldo": 1 << 26}
    assert attend(**a) == 2 and b"attention_cache4" in lcu.lib.lcu_last_error()


def test_beam_workspaces_of_sizes_that_are_refused():
    b = lcu.lib.lcu_beam_select_workspace
    assert b(1, 33, 100, 4) == 0 and b(1, 4, (1 << 24) + 1, 4) == 0 and b(1, 4, 100, 65) == 0 and b(2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1) == 0
    assert b(1, 32, 1 << 24, 64) > 0


def test_calls_from_several_threads_look_for_a_device():
    """Each thread gets its own status and message."""
    if lcu.lib.lcu_device_count() > 0:
        pytest.skip("a GPU is present: these addresses are none")
    from concurrent.futures import ThreadPoolExecutor

    def one(i):
        if i % 2:
            return attend(m=0), lcu.lib.lcu_last_error()
        return append(), lcu.lib.lcu_last_error()

    with ThreadPoolExecutor(8) as pool:
        for i, (rc, words) in enumerate(pool.map(one, range(400))):
            assert (rc == 2 and b"0 rows" in words) if i % 2 else (rc == 1 and b"no CUDA device" in words)
