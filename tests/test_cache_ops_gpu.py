"""GPU tests of the cache operators against the plain 64-bit implementations of
cache_ops_reference.py: words, codes, lengths and positions bit for bit, weights within
the tolerance derived there; slots nobody names are left alone."""
import numpy as np
import pytest
import torch

from cache_ops_reference import codes, evict, key_weights, key_weights_tolerance, make_table, place, rotate, words
from hyperion_b200 import glue

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
i32 = torch.int32


def u32(t):
    return t.cpu().numpy().view(np.uint32)


def gpu(x):
    if isinstance(x, np.ndarray):
        x = torch.from_numpy(x.view(np.int32) if x.dtype == np.uint32 else x.copy())
    return None if x is None else x.to(DEV)


def errors(h):
    return h.read_device_errors(DEV, clear=True)


# ---------------------------------------------------------------------------
# rope_cache_write
# ---------------------------------------------------------------------------
def _write_case(T, Hq, Hk, D, dtype, rot, layout, block, nb, batch, seq_q=1, slots="none", q_idx=False, scales="head",
                seed=0, strided=False, max_pos=500, x=None):
    g = torch.Generator().manual_seed(seed)
    cap, rows = block * nb, batch * Hk
    if x is None:
        x = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(dtype)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]
    # distinct (sequence, slot) pairs
    pairs = torch.randperm(batch * min(cap, seq_q if seq_q > 1 else cap), generator=g)[:T]
    width = min(cap, seq_q if seq_q > 1 else cap)
    seq, slot = (pairs // width).to(i32), (pairs % width).to(i32)
    if seq_q == 1:
        seq = torch.arange(T, dtype=i32)  # one query row per sequence
    pos = slot.clone() if slots == "none" else torch.randint(0, max_pos, (T,), generator=g).to(i32)
    sl = None
    if slots == "token":
        sl = slot
    elif slots == "head":
        sl = torch.stack([(slot + h) % cap for h in range(Hk)], 1).to(i32).contiguous()
    qi = slot.clone() if q_idx else None
    table = make_table(rows, nb, seed + 1) if block < cap else None
    pool = rows * nb * block
    rope = glue.rope_table(max(max_pos, cap), rot) if rot else None
    scale = {"tensor": torch.tensor([0.013]), "head": torch.rand(Hk, generator=g) * 0.01 + 0.005,
             "slot": torch.rand(pool, generator=g) * 0.01 + 0.005}[scales]
    return dict(q=q, k=k, v=v, seq=seq, pos=pos, rope=rope, table=table, block=block, nb=nb, scale=scale, layout=layout,
                seq_q=seq_q, q_idx=qi, slots=sl, batch=batch, strided=strided)


def _write_expected(c, sentinel):
    T, Hq, D = c["q"].shape
    Hk = c["k"].shape[1]
    rows, cap = c["batch"] * Hk, c["block"] * c["nb"]
    pool = rows * cap
    qw = np.full((c["batch"] * Hq * c["seq_q"], D // 32), sentinel, np.uint32)
    kw = np.full((pool, D // 32), sentinel, np.uint32)
    vc = np.full((pool, D), sentinel & 0xFF, np.uint8)
    sp = np.full((rows, cap), -7, np.int32)
    table = None if c["table"] is None else c["table"].numpy()
    rope = None if c["rope"] is None else c["rope"].numpy().astype(np.float64)
    turn = lambda x, p: x if rope is None else rotate(x, rope[p], c["layout"])  # noqa: E731
    q, k = c["q"].double().numpy(), c["k"].double().numpy()
    for i in range(T):
        b, p = int(c["seq"][i]), int(c["pos"][i])
        qi = int(c["q_idx"][i]) if c["q_idx"] is not None else (0 if c["seq_q"] == 1 else p)
        for h in range(Hq):
            qw[(b * Hq + h) * c["seq_q"] + qi] = words(turn(q[i, h], p) >= 0)
        for h in range(Hk):
            s = p if c["slots"] is None else int(c["slots"][i] if c["slots"].dim() == 1 else c["slots"][i, h])
            at = place(table, c["block"], c["nb"], b * Hk + h, s)
            n = c["scale"].numel()
            sc = c["scale"][0 if n == 1 else at if n == pool else (b * Hk + h) % n]
            kw[at], vc[at], sp[b * Hk + h, s] = words(turn(k[i, h], p) >= 0), codes(c["v"][i, h], sc), p
    return qw, kw, vc, sp


def _write_run(h, c, sentinel, stream=None):
    T, Hq, D = c["q"].shape
    Hk = c["k"].shape[1]
    rows, cap = c["batch"] * Hk, c["block"] * c["nb"]
    if c["strided"]:  # slices of a fused projection, at an odd element offset
        both = torch.cat([c["q"], c["k"], c["v"]], 1)
        big = torch.zeros(both.numel() + 1, dtype=both.dtype, device=DEV)[1:].view(both.shape)
        big.copy_(both)
        q, k, v = big[:, :Hq], big[:, Hq:Hq + Hk], big[:, Hq + Hk:]
    else:
        q, k, v = (c[n].contiguous().to(DEV) for n in "qkv")
    qw = torch.full((c["batch"] * Hq * c["seq_q"], D // 32), 0, dtype=i32, device=DEV)
    qw.fill_(np.uint32(sentinel).view(np.int32).item())
    kw = torch.full((rows * cap, D // 32), np.uint32(sentinel).view(np.int32).item(), dtype=i32, device=DEV)
    vc = torch.full((rows * cap, D), sentinel & 0xFF, dtype=torch.uint8, device=DEV)
    sp = torch.full((rows, cap), -7, dtype=i32, device=DEV)
    args = (q, k, v, gpu(c["seq"]), gpu(c["pos"]), gpu(c["rope"]), gpu(c["table"]), c["block"], c["nb"], gpu(c["scale"]), qw, kw, vc)
    kw_args = dict(layout=c["layout"], seq_q=c["seq_q"], q_idx=gpu(c["q_idx"]), slots=gpu(c["slots"]), slot_positions=sp)
    h.rope_cache_write(*args, **kw_args)
    return (qw, kw, vc, sp), (args, kw_args)


def _write_check(h, c, err=0):
    errors(h)
    got, _ = _write_run(h, c, 0xA5A5A5A5)
    assert errors(h) == err
    want = _write_expected(c, 0xA5A5A5A5)
    for name, x, y in zip(("Q words", "K words", "V codes", "positions"), got, want):
        x = x.cpu().numpy()
        x = x.view(np.uint32) if y.dtype == np.uint32 else x
        assert np.array_equal(x, y), (name, np.argwhere(x != y)[:5])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D, rot", [(128, 128), (128, 64), (128, 2), (128, 38), (256, 256), (256, 64), (256, 250), (128, 0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_rope_write_types_and_rotary_dims(hyperion, dtype, D, rot, layout):
    _write_check(hyperion, _write_case(13, 4, 2, D, dtype, rot, layout, 16, 3, 13, seed=D + rot))


@pytest.mark.parametrize("T, Hq, Hk, block, nb, slots, scales, strided", [
    (1, 1, 1, 1, 1, "none", "tensor", False),
    (1, 32, 8, 16, 8, "token", "head", True),
    (7, 6, 2, 20, 3, "head", "slot", True),
    (33, 8, 8, 128, 2, "token", "slot", False),
    (40, 3, 1, 64, 1, "head", "head", True),  # one page a row: contiguous
    (257, 4, 4, 8, 5, "none", "head", False),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rope_write_layouts_slots_and_strides(hyperion, T, Hq, Hk, block, nb, slots, scales, strided, dtype):
    _write_check(hyperion, _write_case(T, Hq, Hk, 128, dtype, 96, "half", block, nb, T, slots=slots, scales=scales,
                                       strided=strided, seed=T))


@pytest.mark.parametrize("q_idx", [False, True])
def test_rope_write_prompt_rows(hyperion, q_idx):
    _write_check(hyperion, _write_case(70, 4, 2, 128, torch.bfloat16, 128, "half", 16, 3, 2, seq_q=48, q_idx=q_idx, seed=5,
                                       slots="token" if q_idx else "none"))


def test_rope_write_sums_next_to_zero_keep_the_exact_sign(hyperion):
    """Sums that cancel to nothing, to one rounding, below the smallest f32, overflow, and NaN."""
    T, D, rot = 6, 128, 128
    c = _write_case(T, 2, 1, D, torch.float32, rot, "half", 16, 2, T, seed=11)
    rope = torch.zeros(32, 2, 64)
    rope[:, 0], rope[:, 1] = 0.70710677, 0.70710677
    rope[:, 0, 1::4] = float(np.nextafter(np.float32(0.70710677), np.float32(1)))  # products one step apart
    rope[:, :, 2::4] = 1.5  # a table with a scale in it: products may overflow
    rope[:, 0, 3::4], rope[:, 1, 3::4] = 1.0, 0.0
    x = torch.randn(T, 4, D, generator=torch.Generator().manual_seed(3))
    x[:, :, 64:] = x[:, :, :64]  # x cos - x sin
    x[1] = 0.0
    x[2, :, :64], x[2, :, 64:] = 3e38, 3e38  # inf - inf of rounded products, exactly 0
    x[2, :, 66::4] = torch.tensor(3.0000001e38)
    x[3] = 1e-38
    x[3, :, :64] = -1.1e-38
    x[3, :, 5::8] = 1e-45
    x[4, :, ::3], x[4, :, 1::3] = float("nan"), float("inf")
    x[5, :, :64], x[5, :, 64:] = -0.0, 0.0
    c.update(q=x[:, :2], k=x[:, 2:3], v=torch.where(x.isfinite(), x, torch.zeros(()))[:, 3:4], rope=rope,
             scale=torch.tensor([1.0]))
    _write_check(hyperion, c)
    for dtype in (torch.bfloat16, torch.float16):
        y = x.clamp(-6e4, 6e4).to(dtype)
        c.update(q=y[:, :2], k=y[:, 2:3], v=torch.zeros_like(y[:, 3:4]), layout="half")
        _write_check(hyperion, c)
    c.update(layout="interleaved")
    _write_check(hyperion, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 0.25, 0.013, 3.0, 1.1, 1e-30, 1e30, float("inf"), -0.7])
def test_rope_write_codes_on_and_next_to_the_borders(hyperion, scale, dtype):
    """V values whose quotient by the scale is a border between two codes, or one step off it."""
    T, D = 64, 128
    c = _write_case(T, 2, 2, D, dtype, 64, "half", 16, 5, T, seed=1)
    grid = torch.cat([torch.arange(0, 18) * 2.0**-10, torch.arange(16, 33)[None].mul(2.0 ** torch.arange(-10, 6)[:, None]).flatten(),
                      torch.tensor([440.0, 448.0, 464.0, 465.0, 500.0, 1e9, float("inf")])]).float()
    v = torch.cat([grid, -grid])[torch.arange(T * 2 * D) % (2 * grid.numel())] * scale
    off = torch.arange(v.numel()) // (2 * grid.numel()) % 5 - 2  # steps of f32 away
    v = torch.where(v.isfinite() & (v != 0), (v.view(torch.int32) + off.to(torch.int32)).view(torch.float32), v)
    c.update(v=torch.nan_to_num(v, nan=0.0, posinf=3e38, neginf=-3e38).to(dtype).view(T, 2, D), scale=torch.tensor([scale]))
    if dtype == torch.bfloat16:
        c["v"] = c["v"].clamp(-3e38, 3e38)
    _write_check(hyperion, c)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype, D, rot, Hq, Hk", [(torch.bfloat16, 128, 128, 32, 8), (torch.float16, 128, 96, 9, 3),
                                                   (torch.float32, 256, 256, 5, 1), (torch.bfloat16, 256, 16, 8, 4),
                                                   (torch.float16, 128, 0, 1, 1)])
def test_rope_write_from_a_fused_projection(hyperion, dtype, D, rot, Hq, Hk, layout):
    """Aligned slices of one tensor; as many tokens as fill the device, and few."""
    h = hyperion
    for T in (3, 700):
        c = _write_case(T, Hq, Hk, D, dtype, rot, layout, 16, 2, T, seed=T + rot)
        both = torch.cat([c["q"], c["k"], c["v"]], 1).to(DEV)
        fused = [both[:, :Hq], both[:, Hq:Hq + Hk], both[:, Hq + Hk:]]
        errors(h)
        want, (args, kw) = _write_run(h, c, 0)
        if T == 3:
            for x, y in zip(want, _write_expected(c, 0)):
                assert np.array_equal(x.cpu().numpy().view(y.dtype)[: y.shape[0]] if y.dtype == np.uint32 else x.cpu().numpy(), y)
        got = [t.clone().zero_() if i < 3 else t.clone().fill_(-7) for i, t in enumerate(want)]
        h.rope_cache_write(*fused, *args[3:10], got[0], got[1], got[2], **{**kw, "slot_positions": got[3]})
        assert errors(h) == 0 and all(torch.equal(a, b) for a, b in zip(got, want))


def test_rope_write_skips_and_flags_what_is_out_of_range(hyperion):
    c = _write_case(8, 4, 2, 128, torch.bfloat16, 64, "half", 16, 3, 8, slots="token", seed=2, max_pos=60)
    h = hyperion
    errors(h)
    (qw0, kw0, vc0, sp0), _ = _write_run(h, c, 0x11111111)
    assert errors(h) == 0

    def again(**change):
        d = {**c, **change}
        (qw, kw, vc, sp), _ = _write_run(h, d, 0x11111111)
        return errors(h), qw, kw, vc, sp

    # a token whose sequence or position does not exist writes nothing, the others all of theirs
    for change in (dict(seq=torch.tensor([0, 1, 2, -1, 4, 5, 6, 7], dtype=i32)),
                   dict(pos=torch.where(torch.arange(8) == 3, 60, c["pos"].long()).to(i32)),
                   dict(pos=torch.where(torch.arange(8) == 3, -1, c["pos"].long()).to(i32))):
        flags, qw, kw, vc, sp = again(**change)
        assert flags == h.DEVERR_BAD_ITEM
        rows = torch.ones(32, dtype=torch.bool)
        rows[12:16] = False  # query rows of sequence 3
        assert torch.equal(qw[rows.to(DEV)], qw0[rows.to(DEV)]) and bool((qw[12:16] == 0x11111111).all())
        assert bool((sp[6:8] == -7).all()) and int((sp >= 0).sum()) == 14
        assert int((vc != 0x11).any(1).sum()) == 14
    # a slot outside the table: Q is still written
    flags, qw, kw, vc, sp = again(slots=torch.where(torch.arange(8) == 3, 48, c["slots"].long()).to(i32))
    assert flags == h.DEVERR_BAD_ITEM and torch.equal(qw, qw0) and int((sp >= 0).sum()) == 14
    # a page outside the pool
    bad = c["table"].clone()
    bad[0, :], bad[1, :] = -1, 1 << 30
    flags, qw, kw, vc, sp = again(table=bad)
    assert flags == h.DEVERR_BAD_BLOCK and torch.equal(qw, qw0) and int((sp >= 0).sum()) == 14
    # a sequence beyond Q and the tables
    flags, qw, kw, vc, sp = again(seq=torch.tensor([0, 1, 2, 99, 4, 5, 6, 7], dtype=i32))
    assert flags == h.DEVERR_BAD_ITEM and bool((qw[12:16] == 0x11111111).all()) and int((sp >= 0).sum()) == 14


@pytest.mark.parametrize("rot", [64, 38])
@pytest.mark.parametrize("seq", [1 << 30, 1 << 29, (1 << 30) + 1, (1 << 31) - 1])
def test_rope_write_of_a_sequence_far_beyond_the_caches(hyperion, seq, rot):
    """Row numbers that pass 64 bits (16 heads x 2^30 rows or pages x the sequence) are out of
    range, not row 0 or a negative one."""
    g = torch.Generator().manual_seed(5)
    H, D, S = 16, 128, 1 << 30
    q, k, v = (torch.randn(1, H, D, generator=g).to(DEV) for _ in range(3))
    rope = glue.rope_table(4, rot).to(DEV)
    qw = torch.full((H, D // 32), 0x11111111, dtype=i32, device=DEV)
    kc, vc = qw.clone(), torch.full((H, D), 0x11, dtype=torch.uint8, device=DEV)
    errors(hyperion)
    one = torch.zeros(1, dtype=i32, device=DEV)
    for seq_q, blocks in ((S, S), (1, S), (S, 1)):
        hyperion.rope_cache_write(q, k, v, one + seq, one, rope, None, 1, blocks, torch.ones(1, device=DEV), qw, kc, vc,
                                  seq_q=seq_q, q_idx=one, slots=one)
        assert errors(hyperion) & hyperion.DEVERR_BAD_ITEM
        assert bool((qw == 0x11111111).all()) and bool((kc == 0x11111111).all()) and bool((vc == 0x11).all())


def test_rope_write_on_another_stream_and_replayed(hyperion):
    c = _write_case(9, 8, 2, 128, torch.float16, 128, "interleaved", 16, 3, 9, seed=4)
    want = _write_expected(c, 0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, (args, kw) = _write_run(hyperion, c, 0)
    s.synchronize()
    assert all(np.array_equal(x.cpu().numpy().view(y.dtype), y) for x, y in zip(got[:3], want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hyperion.rope_cache_write(*args, **kw)
    for t in got[:3]:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert all(np.array_equal(x.cpu().numpy().view(y.dtype), y) for x, y in zip(got[:3], want))


def test_rope_write_of_no_tokens_launches_nothing(hyperion):
    c = _write_case(1, 2, 1, 128, torch.bfloat16, 64, "half", 16, 2, 1)
    got, (args, kw) = _write_run(hyperion, c, 0)
    before = [t.clone() for t in got]
    empty = [t[:0] for t in args[:5]]
    hyperion.rope_cache_write(*empty, *args[5:], **{k: v for k, v in kw.items() if k != "slots"})
    assert all(torch.equal(a, b) for a, b in zip(got, before))


# ---------------------------------------------------------------------------
# accumulate_key_weights
# ---------------------------------------------------------------------------
def _weights_case(lens, Hk, group, D=128, block=16, nb=None, seq_q=1, seed=0, ld=None, pool_extra=0):
    g = torch.Generator().manual_seed(seed)
    ctx = np.repeat(np.array(lens, np.int32), Hk)
    nb = nb or max(1, -(-max(lens) // block))
    rows = ctx.size
    rng = np.random.default_rng(seed)
    return dict(q=rng.integers(0, 2**32, (rows * group * seq_q, D // 32), dtype=np.uint32),
                k=rng.integers(0, 2**32, (rows * nb * block + pool_extra, D // 32), dtype=np.uint32), ctx=ctx,
                table=make_table(rows, nb, seed).numpy(), block=block, nb=nb, seq_q=seq_q, group=group, D=D,
                w=torch.rand(rows, ld or nb * block, generator=g).numpy())


def _weights_check(h, c, causal=False, first=None, n_q=None, decay=1.0, inv=None, in_place=False, err=0):
    D = c["D"]
    inv = 1 / np.sqrt(D) if inv is None else inv
    n_q = n_q or c["seq_q"]
    w = gpu(c["w"])
    out = w if in_place else torch.full_like(w, -3.0)
    errors(h)
    args = (gpu(c["q"]), gpu(c["k"]), gpu(c["ctx"]), gpu(c["table"]), w, c["seq_q"], D, c["block"], c["nb"], inv, causal)
    kw = dict(kv_group=c["group"], q_first=gpu(first), n_q=n_q, decay=decay, out=out)
    assert h.accumulate_key_weights(*args, **kw) is out
    assert errors(h) == err
    got = out.cpu().double().numpy()
    want = key_weights(c["q"], c["k"], c["ctx"], c["table"], c["block"], c["nb"], c["seq_q"], inv, causal, c["group"], first,
                       n_q, decay, c["w"])
    for r, n in enumerate(c["ctx"]):
        n = max(0, min(int(n), c["block"] * c["nb"]))
        tol = key_weights_tolerance(n, c["group"] * n_q, inv, D)
        # a weight at the clamp may be as small as the smallest f32: one of those beside the relative tolerance
        bound = tol * (np.abs(want[r, :n]) + abs(decay) * np.abs(c["w"][r, :n])) + 1.2e-38
        off = np.abs(got[r, :n] - want[r, :n])
        assert np.all(off <= bound), (r, n, np.argmax(off - bound), off.max(), bound.min())
        rest = c["w"][r, n:] if in_place else -3.0
        assert np.array_equal(got[r, n:], np.broadcast_to(np.asarray(rest, np.float64), got[r, n:].shape))
    if not in_place:
        assert np.array_equal(w.cpu().numpy(), c["w"])
        first_bits = out.clone()
        out.fill_(-3.0)
        h.accumulate_key_weights(*args, **kw)
        assert torch.equal(out, first_bits)  # the same inputs, the same bits
    return args, kw


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 16])
@pytest.mark.parametrize("D", [128, 256])
def test_weights_decode_rows(hyperion, group, D):
    _weights_check(hyperion, _weights_case([0, 1, 2, 31, 33, 700], 2, group, D, seed=group))


@pytest.mark.parametrize("block", [1, 8, 16, 20, 64, 128, 1000])
def test_weights_page_sizes(hyperion, block):
    _weights_check(hyperion, _weights_case([999, 515, 16], 1, 4, block=block, nb=-(-1000 // block), seed=block), decay=0.9)


@pytest.mark.parametrize("lens, group", [([4095], 4), ([4097, 8193, 5], 4), ([20011], 2), ([70000], 8), ([33000, 1], 1)])
def test_weights_long_rows(hyperion, lens, group):
    c = _weights_case(lens, 1, group, block=64, seed=sum(lens))
    _weights_check(hyperion, c, in_place=len(lens) == 1)


@pytest.mark.parametrize("n_q", [2, 3, 17, 64, 100])
@pytest.mark.parametrize("group, D", [(1, 128), (4, 128), (3, 256)])
def test_weights_causal_windows(hyperion, n_q, group, D):
    lens = [1, 5, 64, 130, 301]
    c = _weights_case(lens, 2, group, D, seq_q=301, seed=n_q)
    # the last n_q rows of each prompt; those before row 0 do not count
    _weights_check(hyperion, c, causal=True, first=(c["ctx"] - n_q).astype(np.int32), n_q=n_q)


def test_weights_whole_causal_prompt_and_windows_past_the_rows(hyperion):
    c = _weights_case([90, 256, 129], 1, 2, seq_q=256, seed=3)
    _weights_check(hyperion, c, causal=True)
    _weights_check(hyperion, c, causal=False, first=np.array([250, -300, 300], np.int32), n_q=40)
    _weights_check(hyperion, c, causal=True, first=np.array([-2147483648, 2147483647, 0], np.int32), n_q=3)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("group, n_q", [(1, 2), (2, 5), (4, 4)])
def test_weights_short_windows_partly_outside_the_rows(hyperion, group, n_q, causal):
    c = _weights_case([33, 2500, 40, 900], 1, group, seq_q=50, seed=n_q)
    for first in ([-1, 48, 0, 20], [-100, 50, -n_q, 49]):
        _weights_check(hyperion, c, causal=causal, first=np.array(first, np.int32), n_q=n_q)


@pytest.mark.parametrize("D, group, n_q, causal", [(128, 4, 70, True), (128, 2, 64, True), (128, 3, 43, False), (256, 5, 60, True)])
def test_weights_windows_over_many_tiles_and_chunks(hyperion, D, group, n_q, causal):
    lens = [5000, 2048, 2049, 300, 129, 4100]
    c = _weights_case(lens, 1, group, D, block=16, seq_q=5000, seed=group)
    first = (c["ctx"] - n_q + (0 if causal else 5000 - c["ctx"])).astype(np.int32)
    _weights_check(hyperion, c, causal=causal, first=first, n_q=n_q, decay=0.5)
    c["table"][0, 7], c["table"][1, 127], c["table"][5, 200] = -1, 1 << 30, -5
    _weights_check(hyperion, c, causal=causal, first=first, n_q=n_q, err=hyperion.DEVERR_BAD_BLOCK)


@pytest.mark.parametrize("D, group, lens", [(128, 1, [1000, 600, 257]), (128, 3, [700, 1, 513]), (256, 2, [900, 256, 301])])
@pytest.mark.parametrize("causal", [True, False])
def test_weights_whole_prompts_of_many_groups_over_many_chunks(hyperion, D, group, lens, causal):
    """Every row of the prompts (n_q left out): up to nine groups of 256 queries, whose
    products follow one another in the same accumulators, over chunks of 256 keys, among them
    chunks that no query of a group sees."""
    c = _weights_case(lens, 1, group, D, seq_q=max(lens), seed=group + D)
    _weights_check(hyperion, c, causal=causal, decay=0.5)
    _weights_check(hyperion, c, causal=causal, in_place=True)


@pytest.mark.parametrize("D", [128, 256])
def test_weights_many_rows_of_short_and_long_contexts(hyperion, D):
    """Enough keys for the blocks of many keys a thread, ends inside and between them."""
    _weights_check(hyperion, _weights_case([2048, 2047, 2049, 1, 0, 4096, 100, 3000] * 20, 1, 4, D, block=16, nb=256, seed=D))
    c = _weights_case([4100] * 8 + [17] * 150, 1, 3, D, block=1000, seed=D)
    c["table"][3, 2], c["table"][5, 0] = -1, 1 << 29
    _weights_check(hyperion, c, err=hyperion.DEVERR_BAD_BLOCK)


@pytest.mark.parametrize("inv", [-0.09, 0.0, 1.0, -3.0, 1e4])
@pytest.mark.parametrize("seq_q", [1, 40])
def test_weights_scales_of_either_sign_and_beyond_the_clamp(hyperion, inv, seq_q):
    _weights_check(hyperion, _weights_case([77, 400], 2, 4, seq_q=seq_q, seed=9), inv=inv)


@pytest.mark.parametrize("inv", [1.0, -3.0, 1e4])
@pytest.mark.parametrize("D, group", [(128, 3), (256, 5)])
@pytest.mark.parametrize("rows", [5, 250])
def test_weights_beyond_the_clamp_over_many_chunks(hyperion, rows, D, group, inv):
    """The two launches of few queries, each chunk's sum relative to its own best score: one key
    a thread (5 rows) and eight (250); lengths inside a chunk, no key, one, and a chunk whose
    pages all lie outside the pool."""
    h = hyperion
    lens = ([2500, 1, 0, 2100, 300] * 50)[:rows]
    c = _weights_case(lens, 1, group, D, block=64, seed=rows + D)
    assert c["block"] * c["nb"] > 2048
    _weights_check(h, c, inv=inv, decay=0.5)
    c["table"][0, : 32 if rows > 5 else 8] = -1
    c["table"][3, 32] = 1 << 30
    _weights_check(h, c, inv=inv, err=h.DEVERR_BAD_BLOCK)
    c = _weights_case(lens[:5] + [2500] * (rows - 5), 1, group, D, block=64, seq_q=2500, seed=D)
    _weights_check(h, c, inv=inv, causal=True, first=(c["ctx"] - 3).astype(np.int32), n_q=3)


@pytest.mark.parametrize("D, inv", [(128, 1.0), (256, -3.0)])
def test_weights_of_causal_windows_beyond_the_clamp(hyperion, D, inv):
    h = hyperion
    c = _weights_case([400, 33, 1, 0, 270], 1, 2, D, seq_q=400, seed=D)
    first = (c["ctx"] - 40).astype(np.int32)
    _weights_check(h, c, inv=inv, causal=True, first=first, n_q=40, decay=0.5)
    c["table"][0, :3], c["table"][4, 16] = -1, 1 << 30
    _weights_check(h, c, inv=inv, causal=True, first=first, n_q=40, err=h.DEVERR_BAD_BLOCK)
    _weights_check(h, c, inv=inv, causal=True, err=h.DEVERR_BAD_BLOCK)  # the first rows see no key


def test_weights_repeated_keys_and_exact_matches(hyperion):
    c = _weights_case([300], 2, 4, seed=1)
    c["k"][::3] = c["q"][0]
    c["k"][1::3] = ~c["q"][0]
    _weights_check(hyperion, c)
    _weights_check(hyperion, c, inv=-0.5)


@pytest.mark.parametrize("seq_q", [1, 70])
def test_weights_bad_pages_and_lengths(hyperion, seq_q):
    h = hyperion
    c = _weights_case([100, 200, 64], 1, 4, seq_q=seq_q, seed=6)
    c["table"][1, 3], c["table"][1, 5], c["table"][2, :] = -1, 1 << 30, 999999
    _weights_check(h, c, err=h.DEVERR_BAD_BLOCK)
    c = _weights_case([100, 200, 64], 1, 4, seq_q=seq_q, seed=6)
    c["ctx"] = np.array([-5, 100000, 64], np.int32)
    _weights_check(h, c, err=h.DEVERR_NEG_CTX | h.DEVERR_CTX_OVERFLOW)


def test_weights_contiguous_rows_and_a_wider_row_stride(hyperion):
    c = _weights_case([50, 123], 2, 4, block=130, nb=1, seed=8, ld=177)
    c["table"] = None
    _weights_check(hyperion, c)
    _weights_check(hyperion, c, in_place=True)


@pytest.mark.parametrize("D, group, n_q", [(128, 2, 128), (128, 4, 100), (256, 3, 100)])
@pytest.mark.parametrize("cycles, stage", [(2_000_000, 0), (2_000_000, 1), (2_000_000, 3), (1, -1)])
def test_weights_of_a_window_whose_waits_run_out(hyperion, D, group, n_q, cycles, stage):
    """No score is read after a wait that ran out: a product that never comes (the wait ends
    after about a millisecond), or a bound too short for any, ends the call with an error flag,
    and the next call is right.  Every block has at least four products but for the last of a
    row, so each stage is met."""
    c = _weights_case([700, 1500], 2, group, D=D, seq_q=n_q)
    kw = dict(causal=True, first=(c["ctx"] - n_q).astype(np.int32), n_q=n_q)
    args, call = _weights_check(hyperion, c, **kw)
    hyperion.debug_fault(cycles, stage)
    hyperion.accumulate_key_weights(*args, **call)
    torch.cuda.synchronize()
    err = errors(hyperion)
    assert err == hyperion.DEVERR_WAIT_TIMEOUT or (stage < 0 and err == 0)
    _weights_check(hyperion, c, **kw)


def test_the_wait_hook_is_consumed_by_one_call_of_the_weights(hyperion):
    c = _weights_case([90], 1, 1)
    args, call = _weights_check(hyperion, c)
    hyperion.debug_fault(2_000_000, 0)
    hyperion.accumulate_key_weights(*args, **call)  # one query: no wait
    assert errors(hyperion) == 0
    _weights_check(hyperion, _weights_case([300], 1, 2, seq_q=64), n_q=64)


def test_weights_of_no_rows(hyperion):
    w = torch.zeros(0, 16, device=DEV)
    z = torch.zeros(0, 4, dtype=i32, device=DEV)
    out = hyperion.accumulate_key_weights(z, torch.zeros(16, 4, dtype=i32, device=DEV), torch.zeros(0, dtype=i32, device=DEV),
                                          None, w, 1, 128, 16, 1, 0.1, False)
    assert out is w


def test_weights_on_two_streams_and_in_two_graphs(hyperion):
    """Calls in flight at once, eager and replayed, share no scratch."""
    cases = [_weights_case([3000, 500], 2, 4, seq_q=s, seed=s) for s in (1, 33)]
    streams = [torch.cuda.Stream() for _ in cases]
    runs = [_weights_check(hyperion, c) for c in cases]
    want = [kw["out"].clone() for _, kw in runs]
    graphs = []
    for args, kw in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            hyperion.accumulate_key_weights(*args, **kw)
        graphs.append(g)
    for turn in range(20):
        for s, g, (args, kw) in zip(streams, graphs, runs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                if turn % 2:
                    g.replay()
                else:
                    hyperion.accumulate_key_weights(*args, **kw)
    torch.cuda.synchronize()
    assert all(torch.equal(kw["out"], w) for (_, kw), w in zip(runs, want))


# ---------------------------------------------------------------------------
# evict_keys
# ---------------------------------------------------------------------------
def _evict_case(lens, D=128, block=16, nb=None, seed=0, ld=None, slot_scale=False, ties=0.1):
    rng = np.random.default_rng(seed)
    ctx = np.array(lens, np.int32)
    rows = ctx.size
    nb = nb or max(1, -(-max(max(lens), 1) // block))
    pool, ld = rows * nb * block, ld or nb * block
    w = (rng.standard_normal((rows, ld)) ** 4).astype(np.float32)
    w[rng.random((rows, ld)) < ties] = 0.0
    pos = np.stack([rng.permutation(2 * ld)[:ld] for _ in range(rows)]).astype(np.int32)
    return dict(k=rng.integers(0, 2**32, (pool, D // 32), dtype=np.uint32), v=rng.integers(0, 256, (pool, D), dtype=np.uint8),
                scale=rng.random(pool, dtype=np.float32) if slot_scale else None, ctx=ctx,
                table=make_table(rows, nb, seed).numpy(), block=block, nb=nb, w=w, pos=pos)


def _evict_check(h, c, keep, sink=0, recent=0, err=0, in_place=True):
    t = {n: gpu(c[n]) for n in ("k", "v", "scale", "ctx", "table", "w", "pos")}
    outs = {} if in_place else dict(context_lens_out=torch.full_like(t["ctx"], -9), weights_out=torch.full_like(t["w"], -9.0),
                                    positions_out=torch.full_like(t["pos"], -9))
    errors(h)
    new = h.evict_keys(t["k"], t["v"], t["ctx"], t["table"], c["block"], c["nb"], t["w"], t["pos"],
                       keep if np.isscalar(keep) else gpu(np.asarray(keep, np.int32)), sink=sink, recent=recent,
                       V_scale=t["scale"], **outs)
    assert errors(h) == err
    k, v, scale, ctx, w, pos = evict(c["k"], c["v"], c["scale"], c["ctx"], c["table"], c["block"], c["nb"], c["w"], c["pos"],
                                     keep, sink, recent)
    if not in_place:
        assert np.array_equal(u32(t["w"]), c["w"].view(np.uint32)) and np.array_equal(t["pos"].cpu().numpy(), c["pos"])
        assert np.array_equal(t["ctx"].cpu().numpy(), c["ctx"])
        for r, n in enumerate(c["ctx"]):
            n = max(0, min(int(n), c["block"] * c["nb"]))
            w[r, n:], pos[r, n:] = -9.0, -9
    w_got, p_got = (t["w"], t["pos"]) if in_place else (outs["weights_out"], outs["positions_out"])
    assert np.array_equal(new.cpu().numpy(), ctx)
    assert np.array_equal(p_got.cpu().numpy(), pos)
    assert np.array_equal(u32(w_got), w.view(np.uint32))
    assert np.array_equal(u32(t["k"]), k)
    assert np.array_equal(t["v"].cpu().numpy(), v)
    if scale is not None:
        assert np.array_equal(t["scale"].cpu().numpy(), scale)


@pytest.mark.parametrize("lens, keep", [([300, 64, 0, 129], 100), ([5000, 900, 4096], 1000), ([40000, 3], 30000)])
@pytest.mark.parametrize("apart", [("weights",), ("positions",), ("context_lens",), ("weights", "context_lens")])
def test_evict_with_some_outputs_in_place(hyperion, lens, keep, apart):
    """Each output by itself is its input or another tensor."""
    h, c = hyperion, _evict_case(lens, block=16, seed=keep)
    t = {n: gpu(c[n]) for n in ("k", "v", "ctx", "table", "w", "pos")}
    of = {"weights": "w", "positions": "pos", "context_lens": "ctx"}
    outs = {n + "_out": torch.full_like(t[of[n]], -9) for n in apart}
    errors(h)
    new = h.evict_keys(t["k"], t["v"], t["ctx"], t["table"], c["block"], c["nb"], t["w"], t["pos"], keep, sink=4, recent=20,
                       **outs)
    assert errors(h) == 0
    k, v, _, ctx, w, pos = evict(c["k"], c["v"], None, c["ctx"], c["table"], c["block"], c["nb"], c["w"], c["pos"], keep, 4, 20)
    assert np.array_equal(u32(t["k"]), k) and np.array_equal(t["v"].cpu().numpy(), v)
    assert np.array_equal(new.cpu().numpy(), ctx)
    for n, want in (("weights", w), ("positions", pos), ("context_lens", ctx)):
        got = outs[n + "_out"] if n in apart else t[of[n]]
        if n in apart:
            assert np.array_equal(t[of[n]].cpu().numpy(), c[of[n]])  # the input stays
            for r, length in enumerate(c["ctx"]):
                if n != "context_lens":
                    want[r, length:] = -9  # and nothing is written beyond the row
        assert np.array_equal(got.cpu().numpy(), want)


LENS = [0, 1, 2, 16, 31, 33, 200, 511]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("keep", [0, 1, 2, 17, 33, 200, 510, 511, 100000])
def test_evict_budgets(hyperion, keep, in_place):
    _evict_check(hyperion, _evict_case(LENS, seed=keep), keep, in_place=in_place)


@pytest.mark.parametrize("sink, recent", [(0, 1), (4, 0), (4, 64), (10, 1000), (2**31 - 1, 0), (0, 2**31 - 1), (100, 100)])
def test_evict_protected_positions(hyperion, sink, recent):
    # protections wider than the budget among them: the protected key at the lowest slot stays
    for keep in (1, 30, 120):
        _evict_check(hyperion, _evict_case(LENS, seed=sink % 97 + recent % 89), keep, sink, recent)


@pytest.mark.parametrize("block, nb", [(1, 600), (20, 30), (64, 10), (128, 5), (600, 1)])
@pytest.mark.parametrize("D, slot_scale", [(128, True), (256, False)])
def test_evict_page_sizes_and_row_budgets(hyperion, block, nb, D, slot_scale):
    c = _evict_case([600, 0, 577, 64, 300], D, block, nb, seed=block, ld=640, slot_scale=slot_scale)
    if nb == 1:
        c["table"] = None
    _evict_check(hyperion, c, [300, 5, 576, -3, 0], 2, 5)
    _evict_check(hyperion, c, [300, 5, 576, 64, 150], 0, 17, in_place=False)


@pytest.mark.parametrize("lens, keep", [([4097], 4096), ([4096, 5000], 2048), ([20000, 3], 777), ([70001], 35000),
                                        ([140000], 4096), ([300000, 17], 299999), ([500000, 3, 1000], 499000)])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_long_rows(hyperion, lens, keep, in_place):
    _evict_check(hyperion, _evict_case(lens, block=64, seed=keep), keep, 4, 100, in_place=in_place)


@pytest.mark.parametrize("capacity", [803200, 820032])
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_capacities_around_the_most_that_sixteen_blocks_hold(hyperion, capacity, in_place):
    """16 blocks a row of 50,208 keys, nearly all their shared memory, and one block a row
    beyond.  Budgets among ties, below the protected keys and above the length; a bad page."""
    h = hyperion
    c = _evict_case([capacity - 31, 700, 0], block=64, nb=capacity // 64, seed=capacity, slot_scale=True)
    _evict_check(h, c, [capacity - 20000, 650, 5], 4, 100, in_place=in_place)  # 10 % of the sums are 0
    c["table"][0, 12000:12050], c["table"][0, 1] = -1, 1 << 30  # pages of sources, one of destinations
    _evict_check(h, c, [5000, 40, 0], 0, 64, err=h.DEVERR_BAD_BLOCK, in_place=in_place)
    _evict_check(h, c, 50, 2, 2**31 - 1, in_place=in_place)  # all protected: nothing moves
    c["w"][0, ::7], c["w"][0, 1::9] = np.nan, -np.inf
    _evict_check(h, c, 700000, 4, 100, err=h.DEVERR_BAD_BLOCK, in_place=in_place)  # among the NaN


def test_evict_ties_infinities_nan_and_signed_zeros(hyperion):
    c = _evict_case([500, 500, 500, 500, 64], seed=5)
    c["w"][0] = 1.0  # every key the same: the lowest slots stay
    c["w"][1, ::2], c["w"][1, 1::2] = 0.0, -0.0  # equal
    c["w"][2, ::5], c["w"][2, 1::5], c["w"][2, 2::5] = np.nan, np.inf, -np.inf
    c["w"][2, 3::5] = -c["w"][2, 3::5]
    c["w"][3] = np.float32(1e-45) * (np.arange(512) % 7)
    c["w"][4] = np.nan
    for keep in (1, 99, 100, 101, 250, 399, 450):
        _evict_check(hyperion, c, keep)
        _evict_check(hyperion, c, keep, 0, 60)


def test_evict_bad_pages_and_lengths(hyperion):
    h = hyperion
    c = _evict_case([200, 200, 150], seed=7)
    c["table"][0, 11], c["table"][1, 0] = -1, 1 << 30  # a page of sources, one of destinations
    _evict_check(h, c, 100, err=h.DEVERR_BAD_BLOCK)
    c = _evict_case([200, 200, 150], seed=7)
    c["ctx"] = np.array([-1, 1 << 30, 150], np.int32)
    _evict_check(h, c, 100, err=h.DEVERR_NEG_CTX | h.DEVERR_CTX_OVERFLOW)


@pytest.mark.parametrize("rows", [1, 3, 150, 700])
def test_evict_row_counts(hyperion, rows):
    rng = np.random.default_rng(rows)
    _evict_check(hyperion, _evict_case(list(rng.integers(0, 130, rows)) if rows > 1 else [130], nb=9, seed=rows), 64, 4, 16)


def test_evict_of_no_rows(hyperion):
    z = torch.zeros(0, dtype=i32, device=DEV)
    out = hyperion.evict_keys(torch.zeros(16, 4, dtype=i32, device=DEV), torch.zeros(16, 128, dtype=torch.uint8, device=DEV), z,
                              None, 16, 1, torch.zeros(0, 16, device=DEV), torch.zeros(0, 16, dtype=i32, device=DEV), 4)
    assert out is z


def test_evict_replayed_and_on_two_streams(hyperion):
    """Two graphs replayed at once: out of place, so that every replay does the same."""
    cases = [_evict_case([5000, 4000, 700], seed=s) for s in (1, 2)]
    runs, graphs, streams = [], [], [torch.cuda.Stream() for _ in cases]
    for c in cases:
        t = {n: gpu(c[n]) for n in ("k", "v", "ctx", "table", "w", "pos")}
        o = dict(context_lens_out=torch.zeros_like(t["ctx"]), weights_out=torch.zeros_like(t["w"]),
                 positions_out=torch.zeros_like(t["pos"]))
        call = lambda t=t, o=o, c=c: hyperion.evict_keys(t["k"], t["v"], t["ctx"], t["table"], c["block"], c["nb"],  # noqa: E731
                                                         t["w"], t["pos"], 1000, sink=4, recent=32, **o)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        runs.append((t, o, call))
        graphs.append(g)
    for turn in range(10):
        for s, g, (_, _, call) in zip(streams, graphs, runs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay() if turn % 2 else call()
    torch.cuda.synchronize()
    for c, (t, o, _) in zip(cases, runs):
        k, v, _, ctx, w, pos = evict(c["k"], c["v"], None, c["ctx"], c["table"], c["block"], c["nb"], c["w"], c["pos"], 1000, 4, 32)
        assert np.array_equal(u32(t["k"]), k) and np.array_equal(t["v"].cpu().numpy(), v)
        assert np.array_equal(o["context_lens_out"].cpu().numpy(), ctx)
        for r, n in enumerate(c["ctx"]):
            assert np.array_equal(o["weights_out"][r, :n].cpu().numpy(), w[r, :n])
            assert np.array_equal(o["positions_out"][r, :n].cpu().numpy(), pos[r, :n])


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("captured", [False, True])
def test_decode_steps_of_a_bounded_cache(hyperion, oracle, captured):
    """A prompt, its cut to the budget by the last rows' weights, then decode steps at the
    budget: write, forward, weights, evict.  Every step's state is checked against the
    plain implementations on the state before it, the forward against the oracle."""
    h = hyperion
    B, Hq, Hk, D, block, nb, budget, S = 2, 8, 2, 128, 16, 6, 40, 80
    group, rows, cap = Hq // Hk, B * Hk, block * nb
    inv = 1 / np.sqrt(D)
    g = torch.Generator().manual_seed(0)
    table = make_table(rows, nb, 3)
    rope = glue.rope_table(200, D)
    scale = torch.rand(Hk, generator=g) * 0.01 + 0.01
    k = torch.zeros(rows * cap, D // 32, dtype=i32, device=DEV)
    v = torch.zeros(rows * cap, D, dtype=torch.uint8, device=DEV)
    w = torch.zeros(rows, cap, device=DEV)
    sp = torch.full((rows, cap), -1, dtype=i32, device=DEV)
    tb, rp, sc = gpu(table), gpu(rope), gpu(scale)
    errors(h)

    # the prompts: lengths 80 and 57
    lens = [S, 57]
    T = sum(lens)
    x = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(torch.bfloat16).to(DEV)
    seq = torch.cat([torch.full((n,), b, dtype=i32) for b, n in enumerate(lens)]).to(DEV)
    pos = torch.cat([torch.arange(n, dtype=i32) for n in lens]).to(DEV)
    qw = torch.zeros(B * Hq * S, D // 32, dtype=i32, device=DEV)
    h.rope_cache_write(x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:], seq, pos, rp, tb, block, nb, sc, qw, k, v, seq_q=S,
                       slot_positions=sp)
    ctx = torch.tensor(lens, dtype=i32, device=DEV).repeat_interleave(Hk)
    h.accumulate_key_weights(qw, k, ctx, tb, w, S, D, block, nb, inv, True, kv_group=group, q_first=ctx - 16, n_q=16)
    assert errors(h) == 0
    want = key_weights(u32(qw), u32(k), ctx.cpu().numpy(), table.numpy(), block, nb, S, inv, True, group,
                       (ctx - 16).cpu().numpy(), 16, 1.0, np.zeros((rows, cap)))
    assert np.all(np.abs(w.cpu().numpy() - want) <= key_weights_tolerance(S, 64, inv, D) * want)
    assert abs(float(w.sum()) - rows * group * 16) < 1e-2  # every query hands out one
    before = [u32(k), v.cpu().numpy(), None, ctx.cpu().numpy(), table.numpy(), block, nb, w.cpu().numpy(), sp.cpu().numpy()]
    assert h.evict_keys(k, v, ctx, tb, block, nb, w, sp, budget, sink=2, recent=8) is ctx
    after = evict(*before, budget, 2, 8)
    assert all(np.array_equal(a, b) for a, b in zip((u32(k), v.cpu().numpy(), ctx.cpu().numpy(), w.cpu().numpy(), sp.cpu().numpy()),
                                                    (after[0], after[1], after[3], after[4], after[5])))

    # decode steps: one token per sequence, at slot length, then length + 1
    wl = glue.build_worklist(torch.ones(B, dtype=i32, device=DEV), Hq)
    x1 = torch.zeros(B, Hq + 2 * Hk, D, dtype=torch.bfloat16, device=DEV)
    ids, p1 = torch.arange(B, dtype=i32, device=DEV), torch.tensor(lens, dtype=i32, device=DEV)
    q1 = torch.zeros(B * Hq, D // 32, dtype=i32, device=DEV)
    o = torch.zeros(B * Hq, D, dtype=torch.float32, device=DEV)
    slots = torch.zeros(B, Hk, dtype=i32, device=DEV)

    def step():
        slots.copy_(ctx.view(B, Hk))
        h.rope_cache_write(x1[:, :Hq], x1[:, Hq:Hq + Hk], x1[:, Hq + Hk:], ids, p1, rp, tb, block, nb, sc, q1, k, v,
                           slots=slots, slot_positions=sp)
        ctx.add_(1)
        h.hyperion_apex_kernel(wl, wl.shape[0], q1, None, k, None, v, sc, ctx, tb, o, 1, D, D // 8, block, nb, inv, False,
                               kv_group=group)
        h.accumulate_key_weights(q1, k, ctx, tb, w, 1, D, block, nb, inv, False, kv_group=group, decay=0.97)
        mid = [t.clone() for t in (k, v, ctx, w, sp)]
        h.evict_keys(k, v, ctx, tb, block, nb, w, sp, budget, sink=2, recent=8)
        p1.add_(1)
        return mid

    if captured:
        state = [t.clone() for t in (k, v, ctx, w, sp, p1)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            torch.cuda.synchronize()
            for t, s in zip((k, v, ctx, w, sp, p1), state):
                t.copy_(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            mid = step()
    for n in range(6):
        x1.copy_(torch.randn(x1.shape, generator=g).to(torch.bfloat16))
        w0, c0, p0 = w.cpu().numpy(), ctx.cpu().numpy(), p1.cpu().numpy()
        if captured:
            graph.replay()
        else:
            mid = step()
        torch.cuda.synchronize()
        k1, v1, c1, w1, s1 = (t.cpu().numpy() for t in mid)
        k1 = k1.view(np.uint32)
        assert np.array_equal(c1, c0 + 1)
        assert all(s1[r, c0[r]] == p0[r // Hk] for r in range(rows))
        want = key_weights(u32(q1), k1, c1, table.numpy(), block, nb, 1, inv, False, group, None, 1, 0.97, w0)
        assert np.all(np.abs(w1 - want) <= key_weights_tolerance(cap, group, inv, D) * want)
        after = evict(k1, v1, None, c1, table.numpy(), block, nb, w1, s1, budget, 2, 8)
        assert np.array_equal(u32(k), after[0]) and np.array_equal(v.cpu().numpy(), after[1])
        assert np.array_equal(ctx.cpu().numpy(), after[3]) and np.array_equal(w.cpu().numpy(), after[4])
        assert np.array_equal(sp.cpu().numpy(), after[5])
        # the forward over the step's cache, in 64 bits
        vf = torch.from_numpy(v1).view(torch.float8_e4m3fn).double().numpy()
        for b in range(B):
            for hd in range(Hq):
                r = b * Hk + hd // group
                at = [place(table.numpy(), block, nb, r, t) for t in range(int(c1[r]))]
                pop = np.unpackbits((u32(q1)[b * Hq + hd][None] ^ k1[at]).view(np.uint8), axis=1).sum(1)
                e = np.exp((D - 2.0 * pop) * inv - ((D - 2.0 * pop) * inv).max())
                ref = (e / e.sum()) @ vf[at] * float(scale[hd // group])
                ok, mx, _ = oracle.tolerance_check(o[b * Hq + hd].cpu().numpy(), ref)
                assert ok, mx
    if not captured:  # an eager step flags on this stream; a replay on the capture's
        assert errors(h) == 0
