"""Beam decoding on the device, through the C ABI, against the definitions in 64 bits
(beam_reference): lane attention over a shared prefix with window and first rows, beam
selection, beam reordering, and the three together.  Rows that a lane does not see hold NaN.
Moved and appended rows are compared bit for bit, picks exactly, scores to half a step of f32
plus the selection's own arithmetic, attention to the bound derived in beam_reference.bound."""
import ctypes as C

import numpy as np
import pytest

import beam_reference as ref
from mynah_tts_b200 import synth
from mynah_tts_b200.backend import Backend, Decoder, MynahB200Error

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
NP = {"f32": np.float32, "f16": np.float16}


@pytest.fixture(scope="module")
def be():
    b = Backend("f32")
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    b.close()


@pytest.fixture(scope="module")
def tiled():
    """A backend that multiplies every shared prefix on the tensor cores."""
    with pytest.MonkeyPatch.context() as m:
        m.setenv("MYNAH_B200_LANE_TILES", "1")
        b = Backend("f32")
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    yield b
    b.close()


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ints(values):
    return dev(np.asarray(values, np.int64).astype(np.uint32).view(np.int32))


class Lanes:
    """A batch of lanes on the device and its copy on the host; what no lane sees is NaN."""

    def __init__(self, be, kind, heads, hw, lengths, capacity, prefix_lengths=(), voices=None, window=0, sinks=0, seed=0,
                 spread=1.0, slots=None, pad=0, spare=0, gap=0, qkv_gap=0, prefix_spare=0):
        r = np.random.default_rng(seed)
        self.be, self.kind, self.heads, self.hw, self.window, self.sinks = be, kind, heads, hw, window, sinks
        self.lengths, self.capacity, self.prefix_lengths = list(lengths), capacity, list(prefix_lengths)
        n, width = len(lengths), heads * hw
        self.n, self.width = n, width
        self.voices = voices if voices is not None else [0 if prefix_lengths else 1 << 20] * n
        self.n_slots = n + spare
        self.slots = slots if slots is not None else list(r.permutation(self.n_slots)[:n])
        self.scale = 1.0 / np.sqrt(hw)
        self.qkv = np.full((n, 3 * width + qkv_gap), np.nan, np.float32)
        self.qkv[:, :3 * width] = spread * r.normal(size=(n, 3 * width))
        # cache rows are `pad` elements apart, slots `gap` rows apart
        self.store = {m: np.full((self.n_slots, capacity + gap, width + pad), np.nan, NP[kind]) for m in "kv"}
        most = max(prefix_lengths, default=0) + prefix_spare
        self.prefix = {m: np.full((len(prefix_lengths), most, width + pad), np.nan, NP[kind]) for m in "kv"}
        for m in "kv":
            for p, rows in enumerate(prefix_lengths):
                self.prefix[m][p, :rows, :width] = spread * r.normal(size=(rows, width))
            for b in range(n):
                if not 0 <= self.slots[b] < self.n_slots:
                    continue
                P, keep = self.prefix_of(b)
                for row in ref.seen(self.lengths[b], P, window, sinks)[1][:-1]:
                    at = ref.place(row, keep, capacity)
                    self.store[m][self.slots[b], at, :width] = spread * r.normal(size=width)
        self.d = {m: dev(self.store[m]) for m in "kv"}
        self.dp = {m: dev(self.prefix[m]) for m in "kv"}
        self.d_qkv, self.d_len = dev(self.qkv), ints(self.lengths)
        self.d_slot, self.d_voice = ints(self.slots), ints(self.voices)
        self.d_plen = ints(self.prefix_lengths) if prefix_lengths else None
        self.out_gap = 4 if qkv_gap else 0
        self.d_out = torch.full((n, width + self.out_gap), 7.0, device="cuda")
        self.live = None
        floats = be.lane_attention_workspace(n, heads, hw, len(prefix_lengths), most)
        self.space = torch.full((floats,), float("nan"), device="cuda")
        self.most, self.pad, self.gap = most, pad, gap

    def prefix_of(self, b):
        P = self.prefix_lengths[self.voices[b]] if self.voices[b] < len(self.prefix_lengths) else 0
        return P, max(0, self.sinks - P) if self.window else 0

    def cache(self):
        row = self.width + self.pad
        return self.be.lane_cache(self.kind, self.d["k"].data_ptr(), self.d["v"].data_ptr(), self.n_slots, self.capacity,
                                  self.width, row_stride=row, slot_stride=row * (self.capacity + self.gap))

    def bind(self, be=None):
        more = {}
        if self.prefix_lengths:
            more = dict(prefixes=len(self.prefix_lengths), prefix_k=self.dp["k"].data_ptr(), prefix_v=self.dp["v"].data_ptr(),
                        prefix_capacity=self.most, prefix_row_stride=self.width + self.pad,
                        prefix_length=self.d_plen.data_ptr(), lane_prefix=self.d_voice.data_ptr())
            more["prefix_stride"] = self.most * more["prefix_row_stride"]
        return (be or self.be).bind_lane_attention(
            self.cache(), lanes=self.n, heads=self.heads, head_width=self.hw, scale=self.scale, qkv=self.d_qkv.data_ptr(),
            qkv_stride=self.qkv.shape[1], length=self.d_len.data_ptr(), slot=self.d_slot.data_ptr(), window=self.window,
            sinks=self.sinks, out=self.d_out.data_ptr(), out_stride=self.width + self.out_gap,
            live=None if self.live is None else self.live.data_ptr(), workspace=self.space.data_ptr(),
            workspace_floats=self.space.numel(), **more)

    def check(self, live=None, skipped=(), appended=True):
        """The device's results against the definition; lanes >= live and `skipped` are untouched."""
        width = self.width
        out = self.d_out.cpu().numpy()
        want_store = {m: self.store[m].copy() for m in "kv"}
        for b in range(self.n):
            if b in skipped or (live is not None and b >= live):
                assert (out[b] == 7.0).all(), b
                continue
            P, _ = self.prefix_of(b)
            voice = self.voices[b]
            pk = self.prefix["k"][voice, :P, :width] if P else np.zeros((0, width), np.float32)
            pv = self.prefix["v"][voice, :P, :width] if P else np.zeros((0, width), np.float32)
            q, k, v = (self.qkv[b, i * width:(i + 1) * width] for i in range(3))
            s = self.slots[b]
            want, spread = ref.lane(q, k, v, want_store["k"][s, :self.capacity, :width], want_store["v"][s, :self.capacity, :width],
                                    self.lengths[b], pk, pv, self.heads, self.scale, self.window, self.sinks)
            fine = np.isfinite(want)
            assert np.array_equal(out[b, :width][~fine], want[~fine], equal_nan=True), (b, self.lengths[b], P)
            off = np.abs(out[b, :width] - np.where(fine, want, 0))
            assert (off[fine] <= spread[fine]).all(), (b, self.lengths[b], P, float((off / spread)[fine].max()))
            assert (out[b, width:] == 7.0).all()
        for m in "kv":
            got = self.d[m].cpu().numpy()
            assert np.array_equal(got, want_store[m], equal_nan=True)
            self.store[m] = want_store[m]


def attend(be, *a, tiles=None, **kw):
    """tiles: whether the prefixes have to go through the tensor cores, a launch of their own."""
    x = Lanes(be, *a, **kw)
    before = be.launch_count
    x.bind()()
    if tiles is not None:
        assert be.launch_count - before == (3 if tiles else 2)
    be.sync()
    x.check()
    return x


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads, hw", [(12, 64), (12, 16), (1, 128), (5, 24), (3, 80), (13, 32), (25, 8), (64, 16), (2, 120)])
def test_head_layouts(be, kind, heads, hw):
    attend(be, kind, heads, hw, [0, 1, 2, 31, 32, 33, 100], 101, prefix_lengths=[19], seed=heads * hw)


@pytest.mark.parametrize("heads, hw", [(3, 4), (7, 12), (1, 100)])
def test_head_widths_of_four_floats(be, heads, hw):
    attend(be, "f32", heads, hw, [0, 5, 40], 41, prefix_lengths=[7], seed=hw)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("lengths, capacity", [([0], 1), ([1], 2), ([257], 520), ([5000], 5001), ([0, 0, 0], 4), ([3, 0, 900, 0, 1], 901)])
def test_own_rows_only(be, kind, lengths, capacity):
    attend(be, kind, 12, 64, lengths, capacity, seed=len(lengths) + capacity, spare=2)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("lanes, prefix", [(1, 1), (3, 217), (16, 130), (17, 127), (40, 128), (64, 257), (65, 64), (130, 1), (129, 300)])
def test_one_prefix_for_all(be, kind, lanes, prefix):
    r = np.random.default_rng(lanes)
    attend(be, kind, 2, 64, list(r.integers(0, 9, lanes)), 9, prefix_lengths=[prefix], seed=lanes + prefix, prefix_spare=3)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("hw", [16, 48, 128])
def test_prefix_with_other_head_widths(be, kind, hw):
    attend(be, kind, 3, hw, [b % 5 for b in range(70)], 6, prefix_lengths=[143], seed=hw)


# the prefixes as tiles: lanes around the 128 rows of one, rows around its blocks of 32 (f32) and 64
# (f16), heads that leave columns of a slab empty and heads of two slabs
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("lanes, prefix, heads, hw", [(8, 1, 3, 64), (31, 4096, 3, 64), (128, 64, 12, 64), (129, 65, 2, 64), (200, 31, 2, 64),
                                                      (97, 2017, 1, 128), (140, 250, 3, 48), (300, 100, 2, 24), (257, 301, 1, 16),
                                                      (130, 500, 1, 72), (64, 1399, 5, 104), (1024, 33, 1, 32)])
def test_prefix_tiles(tiled, kind, lanes, prefix, heads, hw):
    r = np.random.default_rng(lanes + hw)
    attend(tiled, kind, heads, hw, [int(n) for n in r.integers(0, 9, lanes)], 9, prefix_lengths=[prefix], seed=lanes + prefix,
           prefix_spare=3, tiles=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("hw", [72, 104, 120, 128])
@pytest.mark.parametrize("prefix", [1, 7, 31, 33, 64, 65])
def test_prefix_tiles_of_wide_heads(tiled, kind, hw, prefix):
    """Heads of two slabs behind few rows, where nothing averages out."""
    attend(tiled, kind, 2, hw, [b % 4 for b in range(37)], 5, prefix_lengths=[prefix], seed=hw + prefix, prefix_spare=1, tiles=True)


@pytest.mark.parametrize("walked", [False, True])
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("lanes, prefix, heads, hw", [(40, 4096, 3, 64), (40, 2017, 1, 128), (130, 500, 1, 72), (64, 1399, 5, 104),
                                                      (24, 33, 3, 120), (24, 3000, 4, 32)])
def test_the_drift_behind_a_prefix(kind, lanes, prefix, heads, hw, walked):
    """All outputs together are as precise as operands of 24 (or 22) bits make them, which the bound of
    a single output cannot tell behind many rows (test_beam_host: what it takes of fewer planes)."""
    with pytest.MonkeyPatch.context() as m:
        m.setenv("MYNAH_B200_LANE_TILES", "0" if walked else "1")
        b = Backend("f32")
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    x = attend(b, kind, heads, hw, [i % 4 for i in range(lanes)], 5, prefix_lengths=[prefix], seed=lanes + hw, tiles=not walked)
    b.close()
    out, off, may = x.d_out.cpu().numpy().astype(np.float64), 0.0, 0.0
    for i in range(0, lanes, 3):
        n, width = x.lengths[i], x.width
        kk, vv = (np.concatenate([x.prefix[m][0, :prefix, :width], x.store[m][x.slots[i], :n + 1, :width]]) for m in "kv")
        a, c = ref.drift(x.qkv[i, :width], kk, vv, heads, x.scale, out[i, :width])
        off, may = off + a, may + c
    assert off <= may, np.sqrt(off / may)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_tiles_of_several_prefixes(tiled, kind):
    """Two of them with more than one tile, one empty, one of a single row, lanes without any."""
    r = np.random.default_rng(8)
    lengths = [600, 0, 1, 190, 63]
    voices = [int(v) for v in r.choice([0, 0, 0, 0, 1, 2, 3, 3, 3, 4, 5], 480)]          # 5: no such prefix
    attend(tiled, kind, 2, 64, [int(n) for n in r.integers(0, 5, 480)], 6, prefix_lengths=lengths, voices=voices, seed=2, tiles=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("window, sinks", [(250, 4), (190, 130), (30, 195), (1, 200), (7, 0)])
def test_tiles_behind_a_window(tiled, kind, window, sinks):
    r = np.random.default_rng(window)
    attend(tiled, kind, 2, 64, [0, 1, 5, 90, 210, 260, 900] + [int(n) for n in r.integers(0, 300, 143)], window + sinks + 1,
           prefix_lengths=[200], window=window, sinks=sinks, seed=window, tiles=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_tiles_with_strides_and_odd_values(tiled, kind):
    """Padded rows, unaligned queries, spare slots; then rows of extreme sizes, infinite and NaN
    rows of one prefix, and a live count."""
    r = np.random.default_rng(3)
    attend(tiled, kind, 2, 64, [b % 4 for b in range(150)], 5, prefix_lengths=[190], pad=8, gap=3, qkv_gap=5, spare=4, prefix_spare=2,
           seed=4, tiles=True)
    for spread in (30.0, 1e-4):
        attend(tiled, kind, 2, 64, [b % 4 for b in range(150)], 5, prefix_lengths=[190], spread=spread, seed=5, tiles=True)
    x = Lanes(tiled, kind, 2, 64, [3] * 300, 4, prefix_lengths=[150, 170], voices=[int(v) for v in r.integers(0, 2, 300)], seed=6)
    # a row that one head of every lane looks away from, far larger than the others
    x.prefix["k"][:, 77] = 0.0
    x.prefix["v"][:, 77, 5] = 30000.0
    x.qkv[:, 0] = 30.0
    x.prefix["k"][:, 77, 0] = -30.0
    # and, in the second prefix, values that are no numbers, which its lanes see
    x.prefix["v"][1, 3, 70] = np.inf
    x.prefix["v"][1, 9, 71] = -np.inf
    x.prefix["k"][1, 169, 64] = -np.inf if kind == "f16" else np.nan
    x.dp, x.d_qkv = {m: dev(x.prefix[m]) for m in "kv"}, dev(x.qkv)
    x.live = ints([299])
    x.bind()()
    tiled.sync()
    x.check(live=299)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_tiles_keep_small_weights(tiled, kind):
    """2,000 rows of weight 2.5e-8 beside one of weight 1 whose value is 0.  All terms of the result
    are positive, so it is off by the roundings of its terms relative to ITSELF (the largest value
    is at most three times the mean, which `bound` already counts)."""
    r = np.random.default_rng(11)
    x = Lanes(tiled, kind, 2, 64, [0] * 40, 2, prefix_lengths=[2001], seed=11)
    x.qkv[:] = 0.0
    x.qkv[:, [0, 64]], x.qkv[:, [128, 192]], x.qkv[:, 256:] = 14.0, -10.0, r.uniform(0.5, 1.5, (40, 128))
    x.prefix["k"][:] = 0.0
    x.prefix["k"][:, 1:, [0, 64]] = -10.0
    x.prefix["v"][:] = r.uniform(0.5, 1.5, x.prefix["v"].shape)
    x.prefix["v"][:, 0] = 0.0
    x.dp, x.d_qkv = {m: dev(x.prefix[m]) for m in "kv"}, dev(x.qkv)
    x.bind()()
    tiled.sync()
    got = x.d_out.cpu().numpy()
    for b in range(0, 40, 13):
        q, k, v = (x.qkv[b, i * 128:(i + 1) * 128] for i in range(3))
        want, _ = ref.lane(q, k, v, *(np.zeros((2, 128), NP[kind]) for _ in "kv"), 0, x.prefix["k"][0], x.prefix["v"][0], 2, 0.125, 0, 0)
        tolerance = 3 * ref.bound(np.float64(17.5), 64, 2002) * want
        assert (np.abs(got[b] - want) <= tolerance).all()
    x.check()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_tiles_keep_small_elements_of_a_query(tiled, kind):
    """One element of a million that every row multiplies by zero."""
    x = Lanes(tiled, kind, 2, 64, [0] * 40, 2, prefix_lengths=[300], seed=12)
    x.qkv[:, [5, 69]], x.qkv[:, [133, 197]] = 1e6, 0.0
    x.prefix["k"][..., [5, 69]] = 0.0
    x.dp, x.d_qkv = {m: dev(x.prefix[m]) for m in "kv"}, dev(x.qkv)
    x.bind()()
    tiled.sync()
    x.check()


def test_the_choice_of_tiles(be, tiled):
    """Long prefixes of many lanes are worth a launch, short ones are walked."""
    r = np.random.default_rng(1)
    attend(be, "f16", 12, 64, [int(n) for n in r.integers(0, 4, 64)], 4, prefix_lengths=[3000], seed=1, tiles=True)
    attend(be, "f32", 12, 64, [int(n) for n in r.integers(0, 4, 64)], 4, prefix_lengths=[217], seed=2, tiles=False)
    attend(tiled, "f32", 2, 64, [1] * 7, 4, prefix_lengths=[40], seed=3, tiles=False)
    attend(tiled, "f32", 2, 64, [1] * 8, 4, prefix_lengths=[40], seed=4, tiles=True)
    attend(tiled, "f32", 2, 64, [1] * 80, 4, seed=5, tiles=False)
    with pytest.MonkeyPatch.context() as m:
        m.setenv("MYNAH_B200_NO_TC", "1")
        simt = Backend("f32")
    simt.set_stream(torch.cuda.current_stream().cuda_stream)
    attend(simt, "f16", 12, 64, [1] * 64, 4, prefix_lengths=[3000], seed=1, tiles=False)
    simt.close()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads, hw", [(8, 96), (6, 128), (12, 128), (4, 80), (8, 64)])
def test_tiles_and_rows_that_share_an_sm_or_follow(tiled, kind, heads, hw):
    """Layouts of which one or two tile CTAs fit on an SM, with or without one of the rows; own rows
    that go on for longer than the tiles, and more blocks than CTAs."""
    r = np.random.default_rng(hw)
    attend(tiled, kind, heads, hw, [int(n) for n in r.integers(0, 700, 40)], 701, prefix_lengths=[900], seed=hw, tiles=True)
    attend(tiled, kind, heads, hw, [int(n) for n in r.integers(0, 4, 200)], 4, prefix_lengths=[1500, 40],
           voices=[int(v) for v in r.integers(0, 3, 200)], seed=heads, tiles=True)


def test_the_choice_of_tiles_for_wide_heads(be):
    """A tile CTA of f32 heads above 64 has an SM to itself: half the blocks at a time."""
    r = np.random.default_rng(2)
    for kind, hw, lanes, prefix, tiles in (("f16", 128, 64, 2000, True), ("f16", 128, 9, 200, False), ("f32", 128, 64, 2000, True),
                                           ("f32", 128, 16, 500, False), ("f32", 96, 40, 2000, True), ("f16", 80, 12, 300, False)):
        attend(be, kind, 6, hw, [int(n) for n in r.integers(0, 4, lanes)], 4, prefix_lengths=[prefix], seed=hw, tiles=tiles)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("lanes, prefixes", [(300, 70), (1024, 1024)])
def test_tiles_of_many_prefixes(tiled, kind, lanes, prefixes):
    """More prefixes than a warp has lanes; most tiles hold a few lanes, some prefixes none."""
    r = np.random.default_rng(prefixes)
    lengths = [int(n) for n in r.integers(0, 40, prefixes)]
    attend(tiled, kind, 1, 32, [b % 3 for b in range(lanes)], 4, prefix_lengths=lengths,
           voices=[int(v) for v in r.integers(0, prefixes, lanes)], seed=lanes, tiles=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_slots_and_prefixes_by_default_and_interleaved_caches(be, tiled, kind):
    """No slot and prefix arrays: lane b in slot b, behind prefix 0.  K and V rows side by side in
    one buffer, the prefix rows those of another slot of it."""
    r = np.random.default_rng(17)
    lanes, heads, hw, capacity, prefix = 20, 2, 32, 24, 17
    width, t = heads * hw, NP[kind]
    both = r.normal(size=(lanes + 1, capacity, 2, width)).astype(t)          # the last slot: the prefix
    qkv = r.normal(size=(lanes, 3 * width)).astype(np.float32)
    lengths = [int(n) for n in r.integers(0, capacity, lanes)]
    for b in (be, tiled):
        d, d_qkv, d_len, d_p = dev(both), dev(qkv), ints(lengths), ints([prefix])
        out = torch.zeros((lanes, width), device="cuda")
        size, row = both.itemsize, 2 * width
        at = d.data_ptr() + lanes * capacity * row * size
        cache = b.lane_cache(kind, d.data_ptr(), d.data_ptr() + width * size, lanes, capacity, width, row_stride=row,
                             slot_stride=capacity * row)
        floats = b.lane_attention_workspace(lanes, heads, hw, 1, prefix)
        space = torch.empty(floats, device="cuda")
        b.lane_attention(cache, lanes=lanes, heads=heads, head_width=hw, scale=-0.3, qkv=d_qkv.data_ptr(), length=d_len.data_ptr(),
                         prefixes=1, prefix_k=at, prefix_v=at + width * size, prefix_capacity=prefix, prefix_row_stride=row,
                         prefix_length=d_p.data_ptr(), out=out.data_ptr(), workspace=space.data_ptr(), workspace_floats=floats)
        b.sync()
        want = both.copy()
        for i in range(lanes):
            q, k, v = (qkv[i, j * width:(j + 1) * width] for j in range(3))
            o, spread = ref.lane(q, k, v, want[i, :, 0], want[i, :, 1], lengths[i], both[lanes, :prefix, 0], both[lanes, :prefix, 1],
                                 heads, -0.3, 0, 0)
            assert (np.abs(out[i].cpu().numpy() - o) <= spread).all()
        assert np.array_equal(d.cpu().numpy(), want)


@pytest.mark.parametrize("live", [0, 1])
def test_no_lane_or_one_in_use(be, tiled, live):
    for b in (be, tiled):
        x = Lanes(b, "f32", 2, 32, [4] * 12, 9, prefix_lengths=[30], seed=18)
        x.live = ints([live])
        x.bind()()
        b.sync()
        x.check(live=live)
        assert all(np.array_equal(x.d[m].cpu().numpy(), x.store[m], equal_nan=True) for m in "kv")


def test_scale_of_zero_weighs_all_rows_alike(be, tiled):
    for b in (be, tiled):
        x = Lanes(b, "f16", 2, 64, [4] * 12, 9, prefix_lengths=[30], seed=19)
        x.scale = 0.0
        x.bind()()
        b.sync()
        x.check()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_several_prefixes_one_empty_and_lanes_without(be, kind):
    r = np.random.default_rng(8)
    voices = [int(v) for v in r.integers(0, 6, 90)]          # 5: no such prefix
    attend(be, kind, 3, 64, [int(n) for n in r.integers(0, 30, 90)], 30, prefix_lengths=[70, 0, 1, 200, 33], voices=voices,
           seed=2)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("lanes", [1, 9, 50])
@pytest.mark.parametrize("window, sinks, prefix", [(1, 0, 0), (1, 3, 0), (7, 0, 5), (7, 4, 5), (7, 9, 5), (64, 4, 0), (33, 2, 100),
                                                   (300, 4, 100), (40, 150, 100)])
def test_window_and_first_rows(be, kind, lanes, window, sinks, prefix):
    r = np.random.default_rng(window * 7 + sinks)
    lengths = [0, 1, window, 5 * window + 3][:lanes] + [int(n) for n in r.integers(0, 12 * window, max(0, lanes - 4))]
    attend(be, kind, 3, 32, lengths, window + sinks + int(r.integers(0, 4)), prefix_lengths=[prefix] if prefix else [],
           window=window, sinks=sinks, seed=window)


def test_window_far_into_a_stream(be):
    x = Lanes(be, "f16", 2, 64, [90001, 1, 12345], 1029, window=1025, sinks=4, seed=3)
    x.bind()()
    be.sync()
    x.check()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_strides(be, kind):
    attend(be, kind, 3, 40, [0, 3, 17, 9] * 9, 18, prefix_lengths=[21, 8], voices=[0, 1] * 18, pad=8, gap=3, qkv_gap=5, spare=4,
           prefix_spare=2, seed=4)


def test_large_and_small_values(be):
    """Scores far beyond exp's range and caches of tiny rows."""
    for spread in (30.0, 1e-4):
        for kind in ("f32", "f16"):
            attend(be, kind, 2, 64, [50, 7] * 20, 51, prefix_lengths=[200], spread=spread, seed=5)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_outliers_keep_the_precision_of_the_other_rows(be, kind):
    """One row of a prefix far larger than the rest and looked away from."""
    x = Lanes(be, kind, 2, 64, [3] * 40, 4, prefix_lengths=[150], seed=6)
    x.prefix["k"][0, 77] = 0.0
    x.prefix["v"][0, 77, 5] = 30000.0
    x.qkv[:, 0] = 30.0                                      # the first head looks away from it
    x.prefix["k"][0, 77, 0] = -30.0
    x.dp = {m: dev(x.prefix[m]) for m in "kv"}
    x.d_qkv = dev(x.qkv)
    x.bind()()
    be.sync()
    x.check()


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_infinite_and_nan_rows_that_are_seen(be, kind):
    """What a lane sees decides its result as the definition does; other lanes are untouched."""
    x = Lanes(be, kind, 2, 32, [6] * 20, 8, prefix_lengths=[40, 40], voices=[0] * 10 + [1] * 10, seed=7)
    x.prefix["v"][1, 3, 4] = np.inf
    x.prefix["k"][1, 5, 40] = np.nan
    x.dp = {m: dev(x.prefix[m]) for m in "kv"}
    x.bind()()
    be.sync()
    x.check()
    out = x.d_out.cpu().numpy()
    assert np.isfinite(out[:10]).all() and np.isinf(out[10:, 4]).all() and np.isnan(out[10:, 32:]).all()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads, hw", [(12, 64), (2, 64), (3, 128), (4, 16)])
def test_an_infinite_value_in_the_last_row(be, kind, heads, hw):
    """Wherever a run of rows ends, its last one counts once."""
    x = Lanes(be, kind, heads, hw, list(range(1, 60)), 70, seed=13)
    for b, n in enumerate(x.lengths):
        x.store["v"][x.slots[b], n - 1, b % x.width] = np.inf
    x.d = {m: dev(x.store[m]) for m in "kv"}
    x.bind()()
    be.sync()
    x.check()


def test_lanes_behind_the_live_count_stay(be):
    for live in (0, 1, 5, 12, 99):
        x = Lanes(be, "f32", 3, 32, [4, 0, 9, 2] * 3, 10, prefix_lengths=[20], seed=9)
        x.live = ints([live])
        x.bind()()
        be.sync()
        x.check(live=live)


def test_full_lanes_and_missing_slots_are_left_out_and_reported(be):
    x = Lanes(be, "f32", 3, 32, [4, 10, 9, 11], 10, slots=[2, 1, 7, 0], spare=0, seed=10)
    x.n_slots = 4
    x.bind()()
    with pytest.raises(MynahB200Error, match="cache is full or its slot"):
        be.sync()
    be.sync()
    x.check(skipped=(1, 2, 3))


def test_a_full_lane_is_no_fault_of_what_runs_behind_it(be):
    """The text encoder and the codec of the same backend read their own status; the lane's report
    waits for the sync."""
    from mynah_tts_b200.backend import Codec, TextEncoder
    other = Backend("f32")
    encoder = TextEncoder(other, synth.add_encoder(None, synth.TINY_ENCODER, seed=3), synth.TINY_ENCODER)
    codec = Codec(other, synth.add_codec(None, synth.TINY_CODEC, seed=4), synth.TINY_CODEC, max_frames=4)
    ids, codes = np.array([1, 2, 3], np.int32), synth.make_codec_codes(synth.TINY_CODEC, 5, 2)
    want, sound = encoder.encode(ids), codec.decode(codes)
    for run, result in ((lambda: encoder.encode(ids), want), (lambda: codec.decode(codes), sound)):
        x = Lanes(other, "f32", 3, 32, [4, 10, 9], 10, seed=10)
        x.bind()()
        assert np.array_equal(run(), result)
        with pytest.raises(MynahB200Error, match="cache is full or its slot"):
            other.sync()
        other.sync()
        x.check(skipped=(1,))
    encoder.close()
    codec.close()
    other.close()


@pytest.mark.parametrize("polls", [0, 1, 3])
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads, hw, lanes, tiles", [(12, 64, 9, "0"), (2, 64, 9, "0"), (1, 128, 1, "0"), (2, 64, 70, "1")])
def test_waits_that_run_out_are_reported(be, kind, heads, hw, lanes, tiles, polls):
    """Waits that give up at once, with warps that share a head's rows and without: the call ends, the
    next sync says so, and the calls behind it are sound.  A few polls may or may not do."""
    x = Lanes(be, kind, heads, hw, [300 + 40 * b % 170 for b in range(lanes)], 500, prefix_lengths=[200], seed=14)
    y = Lanes(be, kind, heads, hw, [300 + 40 * b % 170 for b in range(lanes)], 500, prefix_lengths=[200], seed=15)
    with pytest.MonkeyPatch.context() as m:
        m.setenv("MYNAH_B200_LANE_TILES", tiles)
        m.setenv("MYNAH_B200_LANE_POLLS", str(polls))
        short = Backend("f32")
    short.set_stream(torch.cuda.current_stream().cuda_stream)
    x.bind(short)()
    try:
        short.sync()
        said = ""
        x.check()
    except MynahB200Error as e:
        said = str(e)
        assert "ran out" in said
    assert said or polls > 0
    short.sync()                                             # said once
    short.close()
    y.bind()()
    be.sync()
    y.check()


@pytest.mark.parametrize("polls", ["", "many", "-1", "3 ", "99999999999999999999"])
def test_a_wait_that_is_no_number_is_the_default(polls):
    with pytest.MonkeyPatch.context() as m:
        m.setenv("MYNAH_B200_LANE_POLLS", polls)
        b = Backend("f32")
    b.set_stream(torch.cuda.current_stream().cuda_stream)
    attend(b, "f32", 2, 64, [300, 0, 40], 301, prefix_lengths=[30], seed=17)
    b.close()


def test_many_lanes(be):
    r = np.random.default_rng(11)
    attend(be, "f16", 1, 32, [int(n) for n in r.integers(0, 12, 1024)], 12, prefix_lengths=[9, 140],
           voices=[int(v) for v in r.integers(0, 2, 1024)], seed=11)


@pytest.mark.parametrize("kind, heads, hw", [("f32", 6, 64), ("f16", 12, 32), ("f32", 12, 128)])
def test_the_largest_rings(be, kind, heads, hw):
    """Layouts whose steps fill the rows' ring, beside the schedule of the most lanes."""
    attend(be, kind, heads, hw, [b % 3 for b in range(1024)], 3, prefix_lengths=[2], seed=16)


def test_offsets_beyond_32_bits(be):
    """Slots more than 2^32 elements into the cache."""
    heads, hw, capacity = 2, 128, 2 ** 17
    width = heads * hw
    slots = 2 ** 32 // (capacity * width) + 2
    k = torch.zeros((slots, capacity, width), dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    r = np.random.default_rng(12)
    n, slot = 70, slots - 1
    rows = {m: r.normal(size=(n, width)).astype(np.float16) for m in "kv"}
    k[slot, :n], v[slot, :n] = dev(rows["k"]), dev(rows["v"])
    qkv = r.normal(size=(1, 3 * width)).astype(np.float32)
    out = torch.empty(1, width, device="cuda")
    floats = be.lane_attention_workspace(1, heads, hw)
    space = torch.empty(floats, device="cuda")
    cache = be.lane_cache("f16", k.data_ptr(), v.data_ptr(), slots, capacity, width)
    d_qkv, d_len, d_slot = dev(qkv), ints([n]), ints([slot])
    be.lane_attention(cache, lanes=1, heads=heads, head_width=hw, scale=0.1, qkv=d_qkv.data_ptr(), length=d_len.data_ptr(),
                      slot=d_slot.data_ptr(), out=out.data_ptr(), workspace=space.data_ptr(), workspace_floats=floats)
    be.sync()
    host = {m: np.concatenate([rows[m], np.zeros((1, width), np.float16)]) for m in "kv"}
    want, spread = ref.lane(*np.split(qkv[0], 3), host["k"], host["v"], n, rows["k"][:0], rows["v"][:0], heads, 0.1, 0, 0)
    assert (np.abs(out.cpu().numpy()[0] - want) <= spread).all()
    assert np.array_equal(k[slot, n].cpu().numpy(), host["k"][n])
    # and the row moves to another slot
    parent, length = ints([0, 0]), ints([n + 1, 0])
    d_slots = ints([slot, 0])
    be.beam_reorder(cache, requests=1, beams=2, slot=d_slots.data_ptr(), parent=parent.data_ptr(), length=length.data_ptr())
    be.sync()
    assert np.array_equal(k[0, :n + 1].cpu().numpy(), host["k"]) and np.array_equal(v[0, :n + 1].cpu().numpy(), host["v"])


def test_captured_calls_follow_lengths_and_run_beside_each_other(be, monkeypatch):
    """Two graphs with workspaces of their own replayed on two streams at once, lengths moved on
    between replays; a step by step run of the same lanes agrees bit for bit."""
    runs = []
    for seed, kind, tiles in ((20, "f32", "0"), (21, "f16", "1")):
        lanes = Lanes(be, kind, 4, 32, [3, 0, 11, 6] * 25, 40, prefix_lengths=[300], seed=seed)
        monkeypatch.setenv("MYNAH_B200_LANE_TILES", tiles)
        other = Backend("f32")
        stream = torch.cuda.Stream()
        other.set_stream(stream.cuda_stream)
        step = lanes.bind(other)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            with torch.cuda.graph(graph, stream=stream):
                step()
        runs.append((lanes, other, stream, graph))
    for _ in range(3):
        for lanes, other, stream, graph in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for lanes, other, stream, graph in runs:
            lanes.check()
            first = lanes.d_out.clone()
            lanes.bind(other)()
            other.sync()
            assert torch.equal(first, lanes.d_out)
            lanes.lengths = [n + 1 for n in lanes.lengths]
            lanes.d_len += 1
            lanes.d_out.fill_(7.0)
            torch.cuda.synchronize()
    for lanes, other, stream, graph in runs:
        graph.reset()
        other.close()


def test_batch_of_one_lane_equals_a_self_attention_step(be):
    """The single-stream operator of the seam on the same rows."""
    x = attend(be, "f32", 12, 64, [200], 256, seed=13)
    k, v = (be.to_device(x.store[m][x.slots[0]][:200]) for m in "kv")
    kk, vv = (be.dev_alloc(256 * 768) for _ in range(2))
    be.copy_dev(kk.ptr, k.ptr, 200 * 768)
    be.copy_dev(vv.ptr, v.ptr, 200 * 768)
    out = be.dev_alloc(768)
    be.self_attention_dev(C.c_void_p(x.d_qkv.data_ptr()), kk, vv, 200, 768, 201, 12, 64, x.scale, out)
    got = be.d2h(out, 768)
    assert np.abs(got - x.d_out.cpu().numpy()[0]).max() < 2e-6
    for b in (k, v, kk, vv, out):
        b.free()


# ------------------------------------------------------------------------------- selection


def run_select(be, logits, score, done, codebook, eos, allow, stride=None, live=None, in_place=False, offset=0):
    requests, beams, vocab = logits.shape
    stride = stride or vocab
    rows = np.full(offset + requests * beams * stride, np.nan, np.float32)
    for i in range(requests * beams):
        rows[offset + i * stride:offset + i * stride + vocab] = logits.reshape(-1, vocab)[i]
    d = dict(logits=dev(rows), score=dev(score.astype(np.float32).reshape(-1)), done=None if done is None else ints(done.reshape(-1)),
             allow=None if allow is None else ints(allow))
    n = requests * beams
    out = dict(score=torch.full((n,), 7.0, device="cuda"), token=ints([7] * n), parent=ints([7] * n), done=ints([7] * n))
    if in_place:
        out["score"] = d["score"]
        out["done"] = d["done"]
    be.beam_select(logits=d["logits"].data_ptr() + 4 * offset, requests=requests, beams=beams, vocab=vocab, logits_stride=stride,
                   codebook_size=codebook, eos_id=eos, allow_eos=None if allow is None else d["allow"].data_ptr(),
                   score=d["score"].data_ptr(), done=None if done is None else d["done"].data_ptr(),
                   live=None if live is None else live.data_ptr(), score_out=out["score"].data_ptr(),
                   token=out["token"].data_ptr(), parent=out["parent"].data_ptr(), done_out=out["done"].data_ptr())
    be.sync()
    return {k: v.cpu().numpy().reshape(requests, beams) for k, v in out.items()}


def check_select(be, logits, score, done, codebook, eos, allow, **kw):
    requests, beams, _ = logits.shape
    got = run_select(be, logits, score, done, codebook, eos, allow, **kw)
    none = np.zeros((requests, beams), np.int64)
    want = ref.select(logits, score, none if done is None else done, codebook, eos,
                      np.ones(requests, np.int64) if allow is None else allow)
    for name, w in zip(("token", "parent", "done"), want[1:]):
        assert np.array_equal(got[name], w), (name, got[name], w)
    # the stored score: half a step of f32, and the sum of exponentials.  Each term is off by one
    # rounding of its argument (at most 2^-24 |x - max|, weighted by exp(x - max) at most 2^-24),
    # one of the product with log2 e, 2^-22 of the approximation, and a thread adds at most
    # ceil(vocab / 256) of them: 2^-21 + vocab / 256 * 2^-24 relative
    fine = np.isfinite(want[0])
    assert np.array_equal(got["score"][~fine], want[0][~fine].astype(np.float32))
    slack = np.abs(want[0][fine]) * 2.0 ** -24 + 2.0 ** -21 + logits.shape[2] / 256 * 2.0 ** -24
    assert (np.abs(got["score"][fine] - want[0][fine]) <= slack).all()


@pytest.mark.parametrize("requests, beams, vocab", [(1, 1, 1), (1, 1, 5), (1, 4, 64), (3, 2, 33), (2, 3, 4095), (1, 1, 9000),
                                                    (1, 2, 20011), (5, 5, 2048), (2, 8, 2048), (1, 16, 2048), (2, 9, 517),
                                                    (1, 16, 3), (7, 12, 1025), (1, 4, 50021), (2, 7, 8192)])
def test_select(be, requests, beams, vocab):
    r = np.random.default_rng(vocab + beams)
    logits = r.normal(0, 2, (requests, beams, vocab)).astype(np.float32)
    score = -20 * r.random((requests, beams))
    codebook = max(1, vocab - 7)
    check_select(be, logits, score, (r.random((requests, beams)) < 0.2).astype(np.int64), codebook, vocab - 1,
                 (r.random(requests) < 0.5).astype(np.int64), stride=vocab + 3, offset=beams % 4)
    check_select(be, logits, score, None, vocab, vocab + 5, None)


@pytest.mark.parametrize("beams", [1, 4, 16])
def test_select_with_only_the_end_allowed(be, beams):
    """No token but eos_id: one candidate a beam; where it is not allowed either, none."""
    r = np.random.default_rng(beams)
    logits, score = r.normal(size=(3, beams, 40)), r.normal(size=(3, beams))
    check_select(be, logits.astype(np.float32), score.astype(np.float32), None, 0, 39, np.array([1, 0, 1]))
    check_select(be, logits.astype(np.float32), score.astype(np.float32), None, 0, 40, None)


@pytest.mark.parametrize("vocab", [4096, 4097, 8192, 8193, 16384, 16385, 32769])
def test_select_around_the_parts_of_a_row(be, vocab):
    """Rows that fit in registers whole or cut in two, four or eight, and the next size; the best
    tokens on both sides of every cut."""
    r = np.random.default_rng(vocab)
    for beams in (1, 2, 4):
        logits = r.normal(size=(2, beams, vocab)).astype(np.float32)
        for cut in range(1, 8):
            at = vocab * cut // 8
            logits[:, :, max(0, at - 2):at + 2] += 6
        check_select(be, logits, r.normal(size=(2, beams)).astype(np.float32), None, vocab, vocab, None)


def test_select_many_requests(be):
    r = np.random.default_rng(3)
    check_select(be, r.normal(size=(5000, 2, 11)).astype(np.float32), r.normal(size=(5000, 2)).astype(np.float32), None, 9, 10,
                 r.integers(0, 2, 5000))


def test_select_in_place_and_first_step(be):
    """Only the first beam is alive, scores and flags are overwritten."""
    r = np.random.default_rng(1)
    logits = r.normal(size=(3, 5, 300)).astype(np.float32)
    score = np.full((3, 5), -np.inf)
    score[:, 0] = 0.0
    check_select(be, logits, score, np.zeros((3, 5), np.int64), 290, 299, np.ones(3, np.int64), in_place=True)


@pytest.mark.parametrize("order", ["equal", "rising", "falling", "steps", "comb"])
def test_select_orders_and_ties(be, order):
    """Equal logits everywhere, sorted logits, and large ones gathered in one thread's pieces, so
    that far more tokens reach the bound than places."""
    for beams, vocab in ((1, 4097), (8, 6000), (16, 3000)):
        i = np.arange(vocab)
        row = {"equal": np.zeros(vocab), "rising": i / 64.0, "falling": -i / 64.0, "steps": np.floor(i / 100.0),
               "comb": np.where(i // 4 % 256 < 2, 5.0 + i % 7, -np.inf)}[order].astype(np.float32)
        logits = np.broadcast_to(row, (2, beams, vocab)).copy()
        score = np.zeros((2, beams))
        score[1] = -np.arange(beams) / 4.0
        check_select(be, logits, score, None, vocab - 1, vocab - 1, np.array([1, 0]))


@pytest.mark.parametrize("beams, vocab", [(2, 2016), (16, 2016), (3, 257), (2, 20011), (9, 20011), (16, 40960)])
def test_select_of_equal_beams_at_every_alignment(be, beams, vocab):
    """Beams with equal rows and scores are equal, wherever their rows begin: the lower one comes
    first, place by place."""
    r = np.random.default_rng(vocab + beams)
    requests = 12 if vocab < 4096 else 2
    for stride in (vocab, vocab + 1, vocab + 2, vocab + 3):
        rows = r.normal(0, 2, (requests, 1, vocab)).astype(np.float32)
        check_select(be, np.repeat(rows, beams, 1), np.repeat(-20 * r.random((requests, 1)), beams, 1), None, vocab, vocab, None,
                     stride=stride, offset=stride % 3)


@pytest.mark.parametrize("beams, vocab", [(3, 61), (8, 2016), (2, 20011), (16, 9001)])
def test_select_of_equal_beams_with_an_end_gaps_and_flags(be, beams, vocab):
    """Equal beams whose end token counts in the sum, whose rows hold NaN and -inf, some of them done, with
    scores and flags overwritten; and finished ones level with a beam that has one token left."""
    r = np.random.default_rng(vocab)
    row = r.normal(0, 2, vocab).astype(np.float32)
    row[r.integers(0, vocab - 8, vocab // 9)] = np.nan
    row[r.integers(0, vocab - 8, vocab // 9)] = -np.inf
    row[vocab - 1] = np.nanmax(row) - 0.5
    logits = np.repeat(np.stack([row, r.permutation(row)])[:, None], beams, 1)
    logits[1, :, vocab - 1] = np.nan
    done = np.zeros((2, beams), np.int64)
    done[:, 1] = 1
    score = np.full((2, beams), -2.5, np.float32)
    for stride in (vocab, vocab + 1):
        check_select(be, logits, score, done, vocab - 7, vocab - 1, np.array([1, 1]), stride=stride, offset=1, in_place=True)
    only = np.full((2, beams, vocab), -np.inf, np.float32)
    only[:, :, 5] = 3.25
    check_select(be, only, score, done, vocab - 7, vocab - 1, np.array([1, 0]), stride=vocab + 3)


@pytest.mark.parametrize("vocab", [2016, 20011])
def test_select_keeps_the_order_of_close_beams(be, vocab):
    """Beams whose continuations are 1e-9 or 4e-10 apart, by their scores (the rows hold the same
    logits in another order, so the log-sums are equal) or by one small logit of a row: the order
    is that of the definition in 64 bits, whose own rounding is below 1e-13."""
    r = np.random.default_rng(vocab)
    for trial in range(8 if vocab < 4096 else 2):
        row = r.normal(0, 2, vocab).astype(np.float32)
        logits = np.stack([row, r.permutation(row)] * 2)[None]
        score = np.float32([[-1e-3, -1e-3 + 1e-9, -2e-3 + 1e-9, -2e-3]])
        if trial % 2:                                        # one of the smallest logits grows: its beam falls by 1.6e-9
            at = np.argsort(logits[0, 2])[vocab // 200]
            whole = np.exp(row.astype(np.float64)).sum()
            logits[0, 2, at] = np.log(np.exp(np.float64(logits[0, 2, at])) + 1.6e-9 * whole)
        best = np.sort(ref.select(logits, score, np.zeros((1, 4), int), vocab, vocab, np.ones(1))[0][0])
        assert np.diff(best).min() > 5e-11                   # the definition itself has no doubt
        check_select(be, logits, score, None, vocab, vocab, None, stride=vocab + 1)


def test_select_of_rows_beyond_the_turns_that_32_bits_sum(be):
    """Equal beams of 300,001 logits, 37 turns of a thread, that rise by 300 along the vocabulary, so
    that the sums' base moves; and rows most of whose threads see nothing, or NaN, for 32 turns."""
    vocab = 300001
    r = np.random.default_rng(9)
    row = (np.arange(vocab) / 1000.0 + r.normal(0, 1, vocab)).astype(np.float32)
    empty = np.where(np.arange(vocab) % 4096 < 5, row, -np.inf).astype(np.float32)
    odd = np.where(np.arange(vocab) % 4096 < 5, row, np.nan).astype(np.float32)
    done = np.zeros((1, 9), np.int64)
    done[0, 2:] = 1
    score = np.full((1, 9), -np.inf)
    score[0, :2] = -3.0
    for x in (row, empty, odd):
        check_select(be, np.repeat(x[None, None], 9, 1), score, done, vocab - 3, vocab - 1, np.array([0]))


def test_select_with_gathered_large_logits(be):
    """All candidates in the pieces of fewer threads than there are places, thousands of them."""
    vocab = 40960
    i = np.arange(vocab)
    row = np.where(i // 4 % 256 < 6, (i * 37 % 1009) / 100.0, -np.inf).astype(np.float32)
    check_select(be, np.broadcast_to(row, (1, 16, vocab)).copy(), np.linspace(0, -3, 16)[None], None, vocab, vocab, None)
    check_select(be, row[None, None], np.zeros((1, 1)), None, vocab, vocab, None)


def test_select_nan_infinite_and_masked_logits(be):
    r = np.random.default_rng(3)
    logits = r.normal(size=(6, 4, 500)).astype(np.float32)
    logits[0, :, ::3] = np.nan
    logits[1, 1] = -np.inf                                   # a beam without a continuation
    logits[2] = np.nan                                       # a request without one
    logits[3, 2, 7] = np.inf                                 # its beam has no finite sum: dead
    logits[4] = np.finfo(np.float32).min                     # masked with the lowest value, all equal
    logits[4, 1, 9] = 0.0
    logits[5, :, 1:] = -np.inf                               # one token each
    score = -r.random((6, 4))
    score[0, 3] = np.nan
    check_select(be, logits, score, None, 490, 499, None)


def test_select_leaves_requests_behind_the_live_count(be):
    r = np.random.default_rng(4)
    logits = r.normal(size=(4, 3, 100)).astype(np.float32)
    score = -r.random((4, 3))
    got = run_select(be, logits, score, None, 100, 100, None, live=ints([2]))
    want = ref.select(logits, score, np.zeros((4, 3), int), 100, 100, np.ones(4))
    assert np.array_equal(got["token"][:2], want[1][:2]) and (got["token"][2:] == 7).all() and (got["score"][2:] == 7).all()
    assert (got["parent"][2:] == 7).all() and (got["done"][2:] == 7).all()


# ------------------------------------------------------------------------------ reordering


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("requests, beams, layers, capacity, width", [(1, 1, 1, 4, 8), (1, 2, 1, 9, 32), (3, 4, 3, 21, 768),
                                                                      (2, 5, 2, 40, 200), (5, 8, 1, 33, 1032), (2, 16, 2, 17, 264),
                                                                      (70, 3, 1, 5, 64)])
def test_reorder(be, kind, requests, beams, layers, capacity, width):
    r = np.random.default_rng(width + beams)
    n = requests * beams
    pad = 8
    k, v = (r.normal(size=(n + 2, layers, capacity, width + pad)).astype(NP[kind]) for _ in range(2))
    slots = r.permutation(n + 2)[:n]
    parent = r.integers(0, beams, (requests, beams))
    if beams > 2:
        parent[0] = np.roll(np.arange(beams), 1)             # a cycle
        parent[-1, 1] = beams + 3                            # not a beam
    length = r.integers(0, capacity + 1, (requests, beams))
    length[0, 0] = capacity + 5                              # a ring that has turned: every row
    dk, dv = dev(k), dev(v)
    row = width + pad
    cache = be.lane_cache(kind, dk.data_ptr(), dv.data_ptr(), n + 2, capacity, width, row_stride=row,
                          slot_stride=layers * capacity * row, layers=layers, layer_stride=capacity * row)
    d_parent, d_length, d_slot, d_out = ints(parent.reshape(-1)), ints(length.reshape(-1)), ints(slots), ints([-1] * n)
    be.beam_reorder(cache, requests=requests, beams=beams, slot=d_slot.data_ptr(), parent=d_parent.data_ptr(),
                    length=d_length.data_ptr(), length_out=d_out.data_ptr())
    be.sync()
    for host, got in ((k, dk), (v, dv)):
        want = host.copy()
        mine = host[slots].reshape(requests, beams, layers, capacity, row)[..., :width]
        moved, new = ref.reorder(mine, parent, length)
        want[slots, ..., :width] = moved.reshape(n, layers, capacity, width)
        assert np.array_equal(got.cpu().numpy(), want)
    assert np.array_equal(d_out.cpu().numpy().reshape(requests, beams), new)


def test_reorder_live_count_missing_slots_and_identity(be):
    r = np.random.default_rng(5)
    k, v = (r.normal(size=(6, 1, 10, 16)).astype(np.float32) for _ in range(2))
    dk, dv = dev(k), dev(v)
    cache = be.lane_cache("f32", dk.data_ptr(), dv.data_ptr(), 6, 10, 16)
    cache.layer_stride = 160
    live, parent, length = ints([1]), ints([0, 0, 1, 0, 1, 0]), ints([4, 4, 4, 9, 9, 9])
    slot = ints([0, 1, 9, 3, 4, 5])                          # the third beam has no slot
    out = ints([-1] * 6)
    be.beam_reorder(cache, requests=2, beams=3, slot=slot.data_ptr(), parent=parent.data_ptr(), length=length.data_ptr(),
                    length_out=out.data_ptr(), live=live.data_ptr())
    be.sync()
    want = k.copy()
    want[1, :, :4] = k[0, :, :4]
    assert np.array_equal(dk.cpu().numpy(), want) and out.cpu().tolist() == [4, 4, 4, -1, -1, -1]
    # nothing to be had from a lane without a slot, and nowhere to put it: lengths stay
    dk = dev(k)
    cache = be.lane_cache("f32", dk.data_ptr(), dv.data_ptr(), 6, 10, 16)
    cache.layer_stride = 160
    parent, length = ints([2, 0, 0, 5, 3, 4]), ints([3, 4, 5, 6, 7, 8])
    be.beam_reorder(cache, requests=2, beams=3, slot=slot.data_ptr(), parent=parent.data_ptr(), length=length.data_ptr(),
                    length_out=out.data_ptr(), live=live.data_ptr())
    be.sync()
    want = k.copy()
    want[1, :, :3] = k[0, :, :3]
    assert np.array_equal(dk.cpu().numpy(), want) and out.cpu().tolist() == [3, 3, 5, -1, -1, -1]
    before = dk.clone()
    parent = ints([0, 1, 2, 0, 1, 2])
    be.beam_reorder(cache, requests=2, beams=3, parent=parent.data_ptr(), length=length.data_ptr())
    be.sync()
    assert torch.equal(before, dk)


def test_decoder_slots_follow_their_beams():
    """Two candidates of one request part, one is picked twice: its history, continued in two
    slots, gives both the hidden row that it gives alone."""
    shape = synth.TINY
    model = synth.make_model(shape, seed=3)
    be = Backend("f32", strict=True)
    dec = Decoder(be, model, capacity=16, slots=4)
    memory = synth.make_memory(shape, seed=5)
    for s in range(4):
        dec.slot_prefill(s, memory)
    r = np.random.default_rng(6)
    rows = r.normal(size=(6, 3, shape.width)).astype(np.float32)
    slots = [2, 0, 3]
    for t in range(4):
        dec.step_batch(slots[:2] if t > 2 else slots, rows[t][:2] if t > 2 else rows[t])
    kept = [dec.slot_read_kv(s) for s in range(4)]
    dec.reorder(slots, [1, 1, 0], beams=3)                   # lanes 0 and 1 continue lane 1, lane 2 lane 0
    assert [dec.slot_length(s) for s in slots] == [4, 4, 4]
    for b, parent in enumerate([1, 1, 0]):
        k, v = dec.slot_read_kv(slots[b])
        assert np.array_equal(k[:, :4], kept[slots[parent]][0][:, :4]) and np.array_equal(v[:, :4], kept[slots[parent]][1][:, :4])
    assert np.array_equal(dec.slot_read_kv(1)[0], kept[1][0])
    out = dec.step_batch(slots, np.repeat(rows[5][:1], 3, 0))
    assert np.array_equal(out[0], out[1]) and not np.array_equal(out[0], out[2])
    for bad in (([0, 0], [0, 1], 2), ([0, 4], [0, 1], 2), ([0, 1], [0, 2], 2)):
        with pytest.raises(MynahB200Error):
            dec.reorder(bad[0], bad[1], beams=bad[2])
    with pytest.raises(ValueError):
        dec.reorder([0, 1, 2], [0, 1, 0], beams=2)
    dec.close()
    be.close()


# ------------------------------------------------------------------------ the three together


def beam_decode(be, frames, requests, beams, window, sinks, as_graph):
    """A beam search whose "model" is a fixed projection of the attended row, on the device."""
    heads, hw, vocab, prefix = 4, 32, 90, 24
    width, n, capacity = heads * hw, requests * beams, (window + sinks + 1 if window else frames)
    r = np.random.default_rng(30)
    lanes = Lanes(be, "f32", heads, hw, [0] * n, capacity, prefix_lengths=[prefix] * requests,
                  voices=[b // beams for b in range(n)], window=window, sinks=sinks, seed=31)
    for m in "kv":
        lanes.store[m][:] = 0.0                              # every row is written before it is seen
    emb = r.normal(size=(vocab, 3 * width)).astype(np.float32)
    head = (r.normal(size=(width, vocab)) * 0.3).astype(np.float32)
    d_emb, d_head = dev(emb), dev(head)
    logits, score = torch.empty(n, vocab, device="cuda"), torch.empty(n, device="cuda")
    token, parent, done, grown = ints([0] * n), ints([0] * n), ints([0] * n), ints([0] * n)
    lanes.d = {m: torch.zeros_like(lanes.d[m]) for m in "kv"}
    first = np.tile(np.array([0.0] + [-np.inf] * (beams - 1), np.float32), requests)
    stream = torch.cuda.Stream()
    other = Backend("f32")
    other.set_stream(stream.cuda_stream)
    attention = lanes.bind(other)
    select = other.bind_beam_select(logits=logits.data_ptr(), requests=requests, beams=beams, vocab=vocab, codebook_size=80,
                                    eos_id=85, score=score.data_ptr(), done=done.data_ptr(), score_out=score.data_ptr(),
                                    token=token.data_ptr(), parent=parent.data_ptr(), done_out=done.data_ptr())
    move = other.bind_beam_reorder(lanes.cache(), requests=requests, beams=beams, slot=lanes.d_slot.data_ptr(),
                                   parent=parent.data_ptr(), length=grown.data_ptr(), length_out=lanes.d_len.data_ptr())

    def step():
        lanes.d_qkv.copy_(d_emb[token.long()])
        attention()
        torch.matmul(lanes.d_out, d_head, out=logits)
        grown.copy_(lanes.d_len + 1)
        select()
        move()

    picked = []
    with torch.cuda.stream(stream):
        score.copy_(dev(first))
        torch.matmul(lanes.d_out, d_head)                    # the library's workspace, before a capture
        if as_graph:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
        for _ in range(frames):
            graph.replay() if as_graph else step()
            stream.synchronize()
            picked.append([x.cpu().numpy().copy() for x in (score, token, parent, done, lanes.d_len)])
    other.sync()
    if as_graph:
        graph.reset()
    other.close()

    # the same search in 64 bits, following the picks that were made (a pick is a border: it has to
    # be the definition's, or as good as it to the precision of the logits)
    tok, sc, dn = np.zeros(n, int), first.astype(np.float64), np.zeros((requests, beams), int)
    history = [[] for _ in range(n)]
    for f in range(frames):
        rows = np.empty((n, width))
        for b in range(n):
            P = lanes.prefix_of(b)[0]
            x = emb[tok[b]]
            history[b] = history[b] + [x]
            pre, own = ref.seen(f, P, window, sinks)
            kk = np.concatenate([lanes.prefix["k"][lanes.voices[b]][pre], np.array([history[b][j][width:2 * width] for j in own])])
            vv = np.concatenate([lanes.prefix["v"][lanes.voices[b]][pre], np.array([history[b][j][2 * width:] for j in own])])
            q, kk, vv = (np.asarray(t, np.float64).reshape(-1, heads, hw) for t in (x[:width], kk, vv))
            w = lanes.scale * np.einsum("qhd,rhd->hr", q, kk)
            w = np.exp(w - w.max(1, keepdims=True))
            rows[b] = np.einsum("hr,rhd->hd", w / w.sum(1, keepdims=True), vv).reshape(-1)
        x = (rows @ head.astype(np.float64)).reshape(requests, beams, vocab)
        want = ref.select(x, sc.reshape(requests, beams), dn, 80, 85, np.ones(requests))
        got = [t.reshape(requests, beams) for t in picked[f]]
        for i in range(requests):
            for place in range(beams):
                assert abs(got[0][i, place] - want[0][i, place]) < 1e-4, (f, i, place)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3]), f
        assert (picked[f][4] == f + 1).all()
        history = [list(history[b // beams * beams + int(p)]) for b, p in enumerate(want[2].reshape(-1))]
        tok, sc, dn = want[1].reshape(-1), want[0].reshape(-1), want[3]
    return picked


@pytest.mark.parametrize("window, sinks", [(0, 0), (9, 30), (5, 2)])
def test_beam_search(be, window, sinks):
    eager = beam_decode(be, 24, 3, 4, window, sinks, as_graph=False)
    graph = beam_decode(be, 24, 3, 4, window, sinks, as_graph=True)
    for a, b in zip(eager, graph):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
