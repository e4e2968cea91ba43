"""Refusals of the drafted-decoding entry points that the host can see (no GPU: every check
comes before the device is touched), and the oracles' own rules."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import drafting
import tsac_cuda

FAKE = 1 << 20  # never read: the calls below are refused on the host


def cache(**changes):
    s = tsac_cuda._PagedCacheStruct()
    for name in ("pool", "tables", "counts", "lengths", "refs"):
        setattr(s, name, FAKE)
    s.layers, s.pages, s.page_size, s.kv_heads, s.head_dim, s.sequences, s.max_pages, s.type = 2, 8, 16, 4, 128, 4, 4, 0
    for name, value in changes.items():
        setattr(s, name, value)
    return s


def strides(*values):
    return (ctypes.c_ssize_t * len(values))(*values)


def refused(status, words):
    assert status == tsac_cuda.ERROR, status
    message = tsac_cuda.library().tsac_cuda_last_error().decode()
    assert words in message, message


BAD_CACHES = [
    (dict(pool=0), "null paged cache buffer"), (dict(refs=0), "null paged cache buffer"),
    (dict(type=2), "bf16 or fp16"), (dict(type=-1), "bf16 or fp16"),
    (dict(page_size=0), "power of two"), (dict(page_size=24), "power of two"), (dict(page_size=2048), "power of two"),
    (dict(layers=0), "layer count"), (dict(pages=0), "page count"), (dict(pages=(1 << 24) + 1), "page count"),
    (dict(kv_heads=3, head_dim=4), "multiple of 8"), (dict(kv_heads=0), "multiple of 8"),
    (dict(kv_heads=1 << 40, head_dim=1 << 40), "multiple of 8"),
    (dict(sequences=0), "sequence count"), (dict(sequences=65537), "sequence count"),
    (dict(max_pages=0), "table width"), (dict(pool=FAKE + 8), "16-byte aligned"),
]


@pytest.mark.parametrize("changes,words", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(changes, words):
    lib, c = tsac_cuda._drafting(), cache(**changes)
    a, s3 = ctypes.addressof(c), strides(1024, 512, 128)
    refused(lib.tsac_cuda_cache_reserve(a, None, FAKE, 2, 1, FAKE, 1 << 20, None, None), words)
    refused(lib.tsac_cuda_cache_fork(a, FAKE, FAKE, 1, None, None), words)
    refused(lib.tsac_cuda_cache_release(a, None, None, 1, None, None), words)
    refused(lib.tsac_cuda_cache_append(a, 0, FAKE, s3, FAKE, s3, None, None, None, 1, 1, None, None), words)
    refused(lib.tsac_cuda_cache_keep(a, None, FAKE, FAKE, None, 2 * FAKE, 1, 1, None, None), words)
    refused(lib.tsac_cuda_cache_compact(a, 2 * FAKE, 3 * FAKE, FAKE, FAKE, 1 << 20, None, None), words)
    refused(lib.tsac_cuda_tree_attention(a, 0, None, FAKE, None, FAKE, s3, FAKE, s3, None, 4, 1, 1, 1.0, FAKE, 1 << 40,
                                         None, None), words)


def test_list_and_scratch_refusals():
    lib, c = tsac_cuda._drafting(), cache()
    a = ctypes.addressof(c)
    big = lib.tsac_cuda_cache_reserve_scratch_bytes(4, 4)
    assert big >= 4 * 4 * 8
    refused(lib.tsac_cuda_cache_reserve(a, None, FAKE, 5, 4, FAKE, 1 << 20, None, None), "more entries")
    refused(lib.tsac_cuda_cache_reserve(a, FAKE, FAKE, 4097, 4, FAKE, 1 << 30, None, None), "too many")
    refused(lib.tsac_cuda_cache_reserve(a, None, None, 4, 4, FAKE, big, None, None), "null argument")
    refused(lib.tsac_cuda_cache_reserve(a, None, FAKE, 4, 0, FAKE, big, None, None), "slots")
    refused(lib.tsac_cuda_cache_reserve(a, None, FAKE, 4, 5, FAKE, 1 << 20, None, None), "slots")
    refused(lib.tsac_cuda_cache_reserve(a, None, FAKE, 4, 4, FAKE, big - 1, None, None), "scratch")
    refused(lib.tsac_cuda_cache_reserve(a, None, FAKE, 4, 4, FAKE + 4, big, None, None), "scratch")
    refused(lib.tsac_cuda_cache_fork(a, None, FAKE, 1, None, None), "null argument")
    refused(lib.tsac_cuda_cache_fork(a, FAKE, FAKE, 4097, None, None), "too many")
    refused(lib.tsac_cuda_cache_release(a, None, None, 5, None, None), "more entries")
    need = lib.tsac_cuda_cache_compact_scratch_bytes(8)
    refused(lib.tsac_cuda_cache_compact(a, 2 * FAKE, 3 * FAKE, FAKE, FAKE, need - 1, None, None), "scratch")
    refused(lib.tsac_cuda_cache_compact(a, FAKE + 4, 3 * FAKE, FAKE, FAKE, need, None, None), "overlap")
    refused(lib.tsac_cuda_cache_compact(a, 2 * FAKE, FAKE + 4, FAKE, FAKE, need, None, None), "overlap")


def test_row_refusals():
    lib, c = tsac_cuda._drafting(), cache()
    a, good = ctypes.addressof(c), strides(1024, 512, 128)

    def append(layer=0, keys=FAKE, ks=good, values=FAKE, vs=good, most=1):
        return lib.tsac_cuda_cache_append(a, layer, keys, ks, values, vs, None, None, None, 1, most, None, None)

    refused(append(layer=2), "layer out of range")
    refused(append(keys=None), "null argument")
    refused(append(ks=strides(1024, 512, 4)), "multiples of 8")
    refused(append(vs=strides(1022, 512, 128)), "multiples of 8")
    refused(append(values=FAKE + 2), "16-byte aligned")
    refused(append(most=0), "row count")
    refused(lib.tsac_cuda_cache_keep(a, None, FAKE, FAKE, None, FAKE + 4, 1, 1, None, None), "overlap")
    refused(lib.tsac_cuda_cache_keep(a, None, FAKE, FAKE, 2 * FAKE + 12, 2 * FAKE, 1, 1, None, None), "overlap")
    refused(lib.tsac_cuda_cache_keep(a, None, FAKE, FAKE, FAKE, FAKE, 1, 1, None, None), "overlap")
    refused(lib.tsac_cuda_cache_keep(a, None, FAKE, FAKE, None, None, 1, 1, None, None), "null argument")
    refused(lib.tsac_cuda_cache_keep(a, None, FAKE, FAKE, None, 2 * FAKE, 1, 0, None, None), "path width")


def test_attention_refusals():
    lib, good = tsac_cuda._drafting(), strides(1024, 512, 128)

    def attend(c=None, layer=0, parents=FAKE, query=FAKE, qs=good, out=FAKE, os=good, heads=4, count=1, nodes=1,
               scale=1.0, scratch=FAKE):
        c = c or cache()
        return lib.tsac_cuda_tree_attention(ctypes.addressof(c), layer, None, parents, None, query, qs, out, os, None,
                                            heads, count, nodes, scale, scratch, 1 << 40, None, None)

    refused(attend(layer=2), "layer out of range")
    refused(attend(parents=None), "null argument")
    refused(attend(c=cache(head_dim=96)), "head_dim of 64 or 128")
    refused(attend(heads=6), "multiple of the key heads")
    refused(attend(heads=0), "multiple of the key heads")
    refused(attend(nodes=0), "node count")
    refused(attend(nodes=65), "node count")
    refused(attend(scale=float("nan")), "scale")
    refused(attend(scale=float("inf")), "scale")
    refused(attend(qs=strides(1024, 510, 128)), "multiples of 8")
    refused(attend(os=strides(1024, 512, 130)), "multiples of 8")
    refused(attend(query=FAKE + 2), "16-byte aligned")
    refused(attend(count=5), "more entries")


def test_verify_refusals():
    lib = tsac_cuda._drafting()

    def verify(target=FAKE, ts=strides(64, 32), draft=None, ds=None, kind=2, tokens=FAKE, nodes=4, vocab=32, token=FAKE):
        return lib.tsac_cuda_draft_verify(target, ts, draft, ds, kind, tokens, FAKE, FAKE, FAKE, None, 1, nodes, vocab,
                                          FAKE, FAKE, token, None, None)

    refused(verify(kind=3), "bf16, fp16 or fp32")
    refused(verify(target=None), "null argument")
    refused(verify(tokens=None), "null argument")
    refused(verify(token=None), "null argument")
    refused(verify(draft=FAKE), "null argument")
    refused(verify(nodes=0), "node count")
    refused(verify(nodes=65), "node count")
    refused(verify(vocab=0), "vocabulary")
    refused(verify(target=FAKE + 2), "aligned to their type")


def test_calls_for_nothing_need_no_buffers():
    """Empty tensors have null addresses: a call for no entry is no error (but still asks for a device)."""
    lib, c = tsac_cuda._drafting(), cache()
    a, s3 = ctypes.addressof(c), strides(1024, 512, 128)
    nothing = tsac_cuda.OK if torch.cuda.is_available() else tsac_cuda.ERROR_DEVICE
    assert lib.tsac_cuda_cache_reserve(a, None, None, 0, 4, FAKE, 1 << 20, None, None) == nothing
    assert lib.tsac_cuda_cache_fork(a, None, None, 0, None, None) == nothing
    assert lib.tsac_cuda_cache_release(a, None, None, 0, None, None) == nothing
    assert lib.tsac_cuda_cache_append(a, 0, None, s3, None, s3, None, None, None, 0, 1, None, None) == nothing
    assert lib.tsac_cuda_cache_keep(a, None, None, None, None, FAKE, 0, 1, None, None) == nothing
    assert lib.tsac_cuda_tree_attention(a, 0, None, None, None, None, s3, None, s3, None, 4, 0, 1, 1.0, FAKE, 1 << 40,
                                        None, None) == nothing
    assert lib.tsac_cuda_draft_verify(None, strides(1, 1), None, None, 2, None, None, None, None, None, 0, 4, 32, None,
                                      None, None, None, None) == nothing


def test_calls_without_a_gpu_fail_loudly():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    lib, c = tsac_cuda._drafting(), cache()
    assert lib.tsac_cuda_cache_release(ctypes.addressof(c), None, None, 4, None, None) == tsac_cuda.ERROR_DEVICE


def test_binding_refuses_tensors_of_another_kind():
    with pytest.raises(tsac_cuda.TsacError, match="pool must be"):
        tsac_cuda.PagedCache(torch.zeros(1, 2, 4, 16, 1, 64, dtype=torch.bfloat16), *[torch.zeros(1)] * 4)
    with pytest.raises(tsac_cuda.TsacError, match="target must be"):
        tsac_cuda.draft_verify(torch.zeros(1, 2, 8), *[torch.zeros(1)] * 4)


def test_oracle_ancestors():
    assert drafting.ancestors([-1, 0, 0, 1, -2, 4, 9], 7) == [[0], [0, 1], [0, 2], [0, 1, 3], [], [5], []]


@pytest.mark.parametrize("with_draft", [False, True])
def test_verification_leaves_the_target_distribution(with_draft):
    """The rule itself, by integration over a grid of coins and draws: one node with two children."""
    p = np.array([0.5, 0.25, 0.125, 0.125])
    q = np.array([0.25, 0.5, 0.125, 0.125])
    rows = np.stack([p] * 3)
    grid = 32  # probabilities are multiples of 1 / 32 of every stage's mass
    got = np.zeros(4)
    points = (np.arange(grid) + 0.5) / grid
    for a in range(4):
        for b in range(4):
            weight = q[a] * q[b] if with_draft else float((a, b) == (1, 2))
            if weight == 0:
                continue
            for u in points:
                for v in points:
                    for r in points:
                        path, token = drafting.verify(rows, [0, a, b], [-1, 0, 0], [0, u, v], r,
                                                      np.stack([q] * 3) if with_draft else None, 3)
                        first = token if len(path) == 1 else [0, a, b][path[1]]
                        got[first] += weight / grid ** 3
    # Each of three stages is off by at most one grid cell of its mass.
    assert np.abs(got - p).max() <= 3 / grid / 2 + 1e-12


@pytest.mark.parametrize("scale", [3e38, -2.5e38])
def test_scales_that_overflow_in_powers_of_two_are_refused(scale):
    lib, c, s3 = tsac_cuda._drafting(), cache(), strides(1024, 512, 128)
    refused(lib.tsac_cuda_tree_attention(ctypes.addressof(c), 0, None, FAKE, None, FAKE, s3, FAKE, s3, None, 4, 1, 1, scale,
                                         FAKE, 1 << 40, None, None), "scale")


@pytest.mark.parametrize("place", ["sequences", "path", "accepted"])
@pytest.mark.parametrize("in_place", [False, True])
def test_new_lengths_over_another_argument_are_refused(place, in_place):
    """Every plane's CTA reads the lists while the first one writes the new lengths."""
    lib = tsac_cuda._drafting()
    c = cache(tables=3 * FAKE, counts=4 * FAKE, lengths=5 * FAKE, refs=6 * FAKE)
    out = c.lengths if in_place else 7 * FAKE
    given = dict(sequences=8 * FAKE, path=9 * FAKE, accepted=10 * FAKE)
    given[place] = out + 12 if place != "path" else out - 4 * (2 * 3 - 1)  # the last of one over an end of the other
    refused(lib.tsac_cuda_cache_keep(ctypes.addressof(c), given["sequences"], given["path"], given["accepted"], None, out, 2, 3,
                                     None, None), "overlap another argument")


@pytest.mark.parametrize("name", ["tables", "counts", "refs"])
def test_new_lengths_over_the_cache_are_refused(name):
    lib = tsac_cuda._drafting()
    c = cache(tables=3 * FAKE, counts=4 * FAKE, lengths=5 * FAKE, refs=6 * FAKE)
    refused(lib.tsac_cuda_cache_keep(ctypes.addressof(c), None, 8 * FAKE, 9 * FAKE, None, getattr(c, name) + 4, 2, 3, None, None),
            "overlap another argument")


@pytest.mark.parametrize("strides_,count,nodes,overlap", [
    ((1024, 512, 128), 4, 2, None), ((128, 2048, 512), 4, 2, None), ((512, 2048, 128), 4, 3, None), ((8, 512, 128), 1, 2, None),
    ((-1024, 512, 128), 4, 2, None), ((0, 512, 128), 4, 2, "output rows"), ((1024, 0, 128), 4, 2, "output rows"),
    ((1024, 512, 0), 4, 2, "output rows"), ((1024, 512, 120), 4, 2, "output rows"), ((1016, 512, 128), 4, 2, "output rows"),
    ((512, 512, 128), 4, 2, "output rows"), ((1024, -504, 128), 4, 2, "output rows"), ((1 << 60, 512, 128), 4, 2, "output rows"),
    ((1024, 512, -128), 4, 2, None), ((0, 0, 128), 1, 1, None)])
def test_outputs_that_overlap_themselves_are_refused(strides_, count, nodes, overlap):
    lib, c = tsac_cuda._drafting(), cache()
    status = lib.tsac_cuda_tree_attention(ctypes.addressof(c), 0, None, FAKE, None, FAKE, strides(1024, 512, 128), 64 * FAKE,
                                          strides(*strides_), None, 4, count, nodes, 1.0, None, 0, None, None)
    if overlap:
        refused(status, "output rows overlap")
    elif torch.cuda.is_available():
        refused(status, "scratch too small")
    else:
        assert status == tsac_cuda.ERROR_DEVICE


@pytest.mark.parametrize("other", [(1024, 512, 256), (2048, 512, 128), (1024, 1024, 128)])
def test_output_in_place_of_the_query_needs_its_strides(other):
    lib, c = tsac_cuda._drafting(), cache()
    for a, b in (((1024, 512, 128), other), (other, (1024, 512, 128))):
        refused(lib.tsac_cuda_tree_attention(ctypes.addressof(c), 0, None, FAKE, None, FAKE, strides(*a), FAKE, strides(*b), None,
                                             4, 2, 2, 1.0, None, 0, None, None), "output")
