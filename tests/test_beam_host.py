"""What the beam decoding entries refuse, and the definitions that the GPU tests compare with.
No GPU: every refusal is decided from sizes, strides, alignment and null pointers before the
backend is used, so a zeroed block stands in for one."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

import beam_reference as ref
from mynah_tts_b200 import capi
from mynah_tts_b200.backend import Backend, Decoder

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STATE = C.create_string_buffer(4096)
A = 1 << 20                        # an aligned address that no refused call touches


def refusal(fn, args, state=STATE):
    err = C.create_string_buffer(capi.ERR_CAP)
    assert fn(state, None if args is None else C.byref(args), err, capi.ERR_CAP) == -1
    return err.value.decode()


def attention(cache=None, **change):
    c = dict(type=capi.F32, dev_k=A, dev_v=A, slots=4, capacity=32, width=128, row_stride=128, slot_stride=4096,
             layers=1, layer_stride=0)
    c.update(cache or {})
    a = dict(lanes=4, heads=2, head_width=64, scale=0.125, dev_qkv=A, qkv_stride=384, dev_length=A, prefixes=1,
             dev_prefix_k=A, dev_prefix_v=A, prefix_capacity=16, prefix_row_stride=128, prefix_stride=2048,
             dev_prefix_length=A, dev_lane_prefix=A, window=0, sinks=0, dev_out=A, out_stride=128, dev_workspace=A,
             workspace_floats=1 << 30)
    a.update(change)
    args = capi.LaneAttentionArgs(**a)
    args.cache = capi.LaneCache(**c)
    return args


@pytest.mark.parametrize("change, cache, message", [
    (dict(lanes=0), {}, "lanes"), (dict(lanes=1025), {}, "lanes"), (dict(heads=0), {}, "heads"),
    (dict(heads=65, head_width=4), dict(width=260, row_stride=260), "heads"),
    (dict(head_width=0), {}, "head_width"), (dict(head_width=66), {}, "head_width"), (dict(head_width=132), {}, "head_width"),
    ({}, dict(type=capi.INT8), "f32 or f16"), ({}, dict(dev_k=None), "empty"), ({}, dict(dev_v=None), "empty"),
    ({}, dict(capacity=0), "empty"), ({}, dict(slots=0), "empty"),
    ({}, dict(dev_k=A + 4), "16-byte"), ({}, dict(dev_v=A + 8), "16-byte"), ({}, dict(row_stride=124), "16-byte"),
    ({}, dict(row_stride=130), "16-byte"), ({}, dict(slot_stride=4098), "16-byte"), ({}, dict(slot_stride=0), "slot_stride"),
    ({}, dict(type=capi.F16, row_stride=132), "16-byte"),
    ({}, dict(width=124, row_stride=128), "heads * head_width"),
    (dict(heads=4, head_width=4, qkv_stride=48), dict(type=capi.F16, width=16, row_stride=16), "16 bytes"),
    (dict(dev_qkv=None), {}, "buffers"), (dict(qkv_stride=383), {}, "buffers"), (dict(dev_length=None), {}, "buffers"),
    (dict(dev_out=None), {}, "buffers"), (dict(out_stride=127), {}, "buffers"), ({}, dict(slots=3), "slots"),
    (dict(dev_prefix_k=None), {}, "prefixes"), (dict(dev_prefix_length=None), {}, "prefixes"),
    (dict(prefix_capacity=0), {}, "prefixes"), (dict(prefixes=1025), {}, "prefixes"),
    (dict(prefix_row_stride=124), {}, "prefix rows"), (dict(dev_prefix_v=A + 4), {}, "prefix rows"),
    (dict(prefixes=2, prefix_stride=0), {}, "prefix rows"), (dict(prefix_stride=2050), {}, "prefix rows"),
    (dict(prefix_capacity=1 << 30), {}, "2^30"), ({}, dict(capacity=(1 << 31) - 1), "2^30"),
    (dict(prefix_capacity=(1 << 28) - 31), {}, "2^30"), (dict(dev_qkv=A + 2), {}, "buffers"), (dict(dev_out=A + 1), {}, "buffers"),
    (dict(window=33), {}, "window"), (dict(window=30, sinks=3), {}, "window"),
    (dict(window=1, sinks=(1 << 64) - 1), {}, "window"),
    (dict(dev_workspace=None), {}, "workspace"), (dict(dev_workspace=A + 4), {}, "workspace"),
    (dict(workspace_floats=64), {}, "workspace"),
])
def test_lane_attention_refuses(change, cache, message):
    said = refusal(capi.lib().mynah_b200_lane_attention, attention(cache, **change))
    assert message in said, said


def test_null_requests_are_refused():
    lib = capi.lib()
    for fn in (lib.mynah_b200_lane_attention, lib.mynah_b200_beam_select, lib.mynah_b200_beam_reorder):
        assert "invalid" in refusal(fn, None)
    assert "invalid" in refusal(lib.mynah_b200_lane_attention, attention(), state=None)


def test_lane_attention_workspace_outside_the_limits_is_zero():
    size = lambda *a: capi.lib().mynah_b200_lane_attention_workspace(STATE, *a)  # noqa: E731
    assert size(4, 2, 64, 0, 0) > 0
    assert size(0, 2, 64, 0, 0) == size(4, 65, 64, 0, 0) == size(4, 2, 130, 0, 0) == 0
    assert size(4, 2, 64, 1, 1 << 31) == 0


def select(**change):
    a = dict(dev_logits=A, requests=2, beams=4, vocab=64, logits_stride=64, codebook_size=60, eos_id=63, dev_score=A,
             dev_score_out=A, dev_token=A, dev_parent=2 * A)
    a.update(change)
    return capi.BeamSelectArgs(**a)


@pytest.mark.parametrize("change", [
    dict(requests=0), dict(beams=0), dict(requests=(1 << 24) + 1), dict(beams=17), dict(vocab=0), dict(vocab=1 << 30, logits_stride=1 << 30),
    dict(codebook_size=65), dict(logits_stride=63), dict(dev_logits=None), dict(dev_score=None), dict(dev_score_out=None),
    dict(dev_token=None), dict(dev_parent=None), dict(dev_parent=A), dict(dev_logits=A + 2)])
def test_beam_select_refuses(change):
    assert refusal(capi.lib().mynah_b200_beam_select, select(**change))


def reorder(cache=None, **change):
    c = dict(type=capi.F32, dev_k=A, dev_v=A, slots=8, capacity=32, width=128, row_stride=128, slot_stride=8192,
             layers=2, layer_stride=4096)
    c.update(cache or {})
    a = dict(requests=2, beams=4, dev_parent=A, dev_length=A, dev_length_out=2 * A)
    a.update(change)
    args = capi.BeamReorderArgs(**a)
    args.cache = capi.LaneCache(**c)
    return args


@pytest.mark.parametrize("change, cache", [
    (dict(requests=0), {}), (dict(requests=65536), dict(slots=1 << 20)), (dict(beams=0), {}), (dict(beams=17), {}),
    (dict(dev_parent=None), {}), (dict(dev_length=None), {}), (dict(dev_length_out=A), {}), ({}, dict(slots=7)),
    ({}, dict(layers=0)), ({}, dict(layers=32768)), ({}, dict(layer_stride=0)), ({}, dict(layer_stride=4098)),
    ({}, dict(width=126)), ({}, dict(dev_k=A + 4))])
def test_beam_reorder_refuses(change, cache):
    assert refusal(capi.lib().mynah_b200_beam_reorder, reorder(cache, **change))


def test_arrays_that_are_not_aligned_are_refused():
    """The kernels read and write them as 32-bit values, which a device faults on elsewhere."""
    lib = capi.lib()
    for fn, make, names in (
            (lib.mynah_b200_lane_attention, attention, "dev_slot dev_length dev_prefix_length dev_lane_prefix dev_live"),
            (lib.mynah_b200_beam_select, select,
             "dev_allow_eos dev_score dev_done dev_live dev_score_out dev_token dev_parent dev_done_out"),
            (lib.mynah_b200_beam_reorder, reorder, "dev_slot dev_parent dev_length dev_length_out dev_live")):
        for name in names.split():
            for off in (1, 2, 3):
                said = refusal(fn, make(**{name: 4 * A + off}))
                assert "4-byte aligned" in said, (name, said)


def test_decoder_reorder_refuses_without_a_decoder():
    err = C.create_string_buffer(capi.ERR_CAP)
    one = (C.c_uint * 1)(0)
    assert capi.lib().mynah_b200_decoder_reorder(None, one, one, 1, 1, err, capi.ERR_CAP) == -1
    assert b"reorder" in err.value


def test_decoder_reorder_refuses_rows_that_are_not_16_byte_pieces():
    """A block of ones instead of a decoder: its width is odd, its slots are plenty; nothing else
    of it may be read before the refusal."""
    decoder, err = C.create_string_buffer(b"\xff" * (1 << 16)), C.create_string_buffer(capi.ERR_CAP)
    two = (C.c_uint * 2)(0, 1)
    assert capi.lib().mynah_b200_decoder_reorder(decoder, two, two, 1, 2, err, capi.ERR_CAP) == -1
    assert b"multiples of 4" in err.value


@pytest.mark.parametrize("slots, parents, beams", [([0, 1], [0, 0], 0), ([0, 1], [0, 0], -1), ([0, 1, 2], [0, 0, 0], 2),
                                                   ([0, 1], [0], 2), ([[0, 1]], [[0, 0]], 2)])
def test_decoder_reorder_refuses_other_shapes(slots, parents, beams):
    with pytest.raises(ValueError, match="requests \\* beams"):
        Decoder.reorder(Decoder.__new__(Decoder), slots, parents, beams)


def test_bound_calls_report_a_refusal():
    be = Backend.__new__(Backend)
    be.lib, be.state = capi.lib(), None
    with pytest.raises(capi.MynahB200Error, match="invalid beam selection"):
        be.beam_select(logits=A, requests=1, beams=1, vocab=4, codebook_size=4, eos_id=4, score=A, score_out=A, token=A,
                       parent=A)


def beam_recipe():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    return re.search(r"## 3b.*?```c\n(.*?)```", text, re.S).group(1)


def test_the_documented_step_compiles(tmp_path):
    """INTEGRATION.md's step against the header, with what it takes from its surroundings declared."""
    source = tmp_path / "step.c"
    source.write_text("""#include "mynah_b200.h"
void project_logits(const float *out, float *logits);
void advance(const unsigned *length, unsigned *grown, size_t n);
void step(void *state, void *k, void *v, void *pk, void *pv, float *qkv, float *out, float *space, float *logits, float *score,
          unsigned *length, unsigned *grown, unsigned *context_length, unsigned *token, unsigned *parent, unsigned *done,
          size_t slots, size_t capacity, size_t width, size_t layers, size_t n, size_t requests, size_t beams, size_t vocab,
          size_t codebook_size, size_t eos_id, size_t context_rows, char *err, size_t cap) {
""" + beam_recipe() + "}\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"),
                    str(source)], check=True)


def test_the_documented_step_moves_the_newest_row():
    """Its order of calls and its lengths, with the definitions in the calls' place: a beam that takes
    another's place goes on from that one's newest row."""
    recipe = beam_recipe()
    calls = re.findall(r"^(\w+)\(", recipe, re.M)
    given = re.search(r"\.dev_length = (\w+), \.dev_length_out = (\w+)", recipe).groups()
    assert given[1] == "length"
    k = np.zeros((1, 2, 1, 8, 1))
    at = {"length": np.array([[3, 3]])}
    for call in calls:
        if call == "mynah_b200_lane_attention":
            k[0, :, 0, 3, 0] = [10.0, 20.0]                  # each lane's new row, behind its three
        elif call == "advance":
            at["grown"] = at["length"] + 1
        elif call == "mynah_b200_beam_reorder":
            k, at["length"] = ref.reorder(k, np.array([[1, 1]]), at[given[0]])
    assert k[0, :, 0, 3, 0].tolist() == [20.0, 20.0] and at["length"].tolist() == [[4, 4]]


# ---- the definitions against cases worked out by hand


def test_seen_rows():
    # prefix 3, own rows 0..4 and the new row 5: joined positions 0..8
    assert ref.seen(5, 3, 0, 0) == ([0, 1, 2], [0, 1, 2, 3, 4, 5])
    assert ref.seen(5, 3, 2, 0) == ([], [4, 5])
    assert ref.seen(5, 3, 2, 2) == ([0, 1], [4, 5])
    assert ref.seen(5, 3, 2, 4) == ([0, 1, 2], [0, 4, 5])
    assert ref.seen(5, 3, 7, 1) == ([0, 2], [0, 1, 2, 3, 4, 5])
    assert ref.seen(5, 3, 100, 4) == ([0, 1, 2], [0, 1, 2, 3, 4, 5])
    assert ref.seen(0, 0, 1, 3) == ([], [0])
    assert [ref.place(r, 2, 6) for r in range(11)] == [0, 1, 2, 3, 4, 5, 2, 3, 4, 5, 2]


def planes(a, n, half=False):
    """The first n 16-bit planes of a: bf16, or f16."""
    left, got = np.asarray(a, np.float64), np.zeros_like(a, dtype=np.float64)
    for _ in range(n):
        if half:
            part = left.astype(np.float16).astype(np.float64)
        else:
            bits = left.astype(np.float32).view(np.uint32).astype(np.uint64)
            part = ((bits + 0x7fff + (bits >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(np.float32).astype(np.float64)
        got, left = got + part, left - part
    return got


@pytest.mark.parametrize("rows, hw", [(2, 128), (33, 72), (500, 72), (1399, 104), (2017, 128), (4096, 64)])
def test_the_drift_that_is_allowed_tells_planes_apart(rows, hw):
    """Results with one operand cut to fewer planes than the kernels keep are refused, whichever it is;
    32-bit arithmetic is not."""
    r = np.random.default_rng(rows)
    lanes, scale = 12, 1.0 / np.sqrt(hw)
    k, v = r.normal(size=(2, rows, hw)).astype(np.float32)
    q = r.normal(size=(lanes, hw)).astype(np.float32)

    def ratio(cut, n, half=False):
        keep = {name: (lambda a, name=name: planes(a, n, half) if name == cut else np.asarray(a, np.float64)) for name in "qkwv"}
        off = may = 0.0
        for b in range(lanes):
            x = scale * keep["k"](k) @ keep["q"](q[b])
            w = np.exp(x - x.max())
            out = keep["w"](w) @ keep["v"](v) / w.sum()
            a, c = ref.drift(q[b], k, v, 1, scale, out)
            off, may = off + a, may + c
        return np.sqrt(off / may)

    for cut in "qkwv":
        assert ratio(cut, 1) > 100 and ratio(cut, 3) < 0.1, cut
        assert ratio(cut, 1, half=True) > 10 and ratio(cut, 2, half=True) < 0.5, cut
        if rows > 2:
            assert ratio(cut, 2) > 1, cut
    off = may = 0.0
    for b in range(lanes):
        x = (np.float32(scale) * q[b]) @ k.T
        w = np.exp(x - x.max())
        a, c = ref.drift(q[b], k, v, 1, scale, (w @ v / w.sum()).astype(np.float64))
        off, may = off + a, may + c
    assert off < may


def test_selection_rules():
    x = np.log(np.array([[[4.0, 2.0, 1.0, 1.0], [1.0, 1.0, 5.0, 1.0]]], np.float32))
    score, token, parent, done = ref.select(x, np.zeros((1, 2), np.float32), np.zeros((1, 2), int), 3, 3, np.array([1]))
    assert token.tolist() == [[2, 0]] and parent.tolist() == [[1, 0]] and np.allclose(score, np.log([[5 / 8, 4 / 8]]))
    # equal scores: the lower beam, then the lower token; eos only where it is allowed
    x = np.zeros((1, 3, 4), np.float32)
    x[0, 2, 3] = 9.0
    score, token, parent, done = ref.select(x, np.zeros((1, 3), np.float32), np.zeros((1, 3), int), 3, 3, np.array([0]))
    assert token.tolist() == [[0, 1, 2]] and parent.tolist() == [[0, 0, 0]] and not done.any()
    # a finished beam goes on as it is; places without a continuation are dead
    x = np.full((1, 3, 4), np.nan, np.float32)
    x[0, 0, 1] = 2.0
    s = np.array([[-1.0, -0.5, -np.inf]], np.float32)
    score, token, parent, done = ref.select(x, s, np.array([[0, 1, 0]]), 3, 3, np.array([1]))
    assert token.tolist() == [[3, 1, 0]] and parent.tolist() == [[1, 0, 2]] and done.tolist() == [[1, 0, 0]]
    assert score.tolist() == [[-0.5, -1.0, -np.inf]]
