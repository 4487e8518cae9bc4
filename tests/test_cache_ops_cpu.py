"""Refusals of the cache operators, in Python and at the C boundary, and the rotary table:
no device is touched."""
import ctypes
import math

import numpy as np
import pytest
import torch

i32, f32 = torch.int32, torch.float32


def _write_args(T=3, Hq=4, Hk=2, D=128, rot=64, pool=64, block=16, nb=2, B=2):
    return dict(Q_new=torch.zeros(T, Hq, D), K_new=torch.zeros(T, Hk, D), V_new=torch.zeros(T, Hk, D),
                seq_ids=torch.zeros(T, dtype=i32), positions=torch.zeros(T, dtype=i32), rope=torch.zeros(8, 2, rot // 2),
                block_tables=None, block_size=block, num_blocks=nb, V_scale=torch.ones(1),
                Q_words=torch.zeros(B * Hq, D // 32, dtype=i32), K_cache=torch.zeros(pool, D // 32, dtype=i32),
                V_cache=torch.zeros(pool, D, dtype=torch.uint8))


@pytest.mark.parametrize("change, match", [
    (dict(Q_new=torch.zeros(3, 4, 128, dtype=torch.float64)), "dtype"),
    (dict(K_new=torch.zeros(3, 2, 128, dtype=torch.float16)), "dtype"),
    (dict(Q_new=torch.zeros(3, 4 * 128)), "n_heads"),
    (dict(V_new=torch.zeros(3, 1, 128)), "n_kv_heads"),
    (dict(Q_new=torch.zeros(2, 4, 128)), "tokens"),
    (dict(Q_new=torch.zeros(3, 4, 256)), "head_dim"),
    (dict(Q_new=torch.zeros(3, 4, 64), K_new=torch.zeros(3, 2, 64), V_new=torch.zeros(3, 2, 64)), "head_dim must be"),
    (dict(Q_new=torch.zeros(3, 0, 128)), "n_heads"),
    (dict(Q_new=torch.zeros(3, 128, 4).transpose(1, 2)), "contiguous"),
    (dict(seq_ids=torch.zeros(3, dtype=torch.int64)), "seq_ids"),
    (dict(positions=torch.zeros(2, dtype=i32)), "positions"),
    (dict(q_idx=torch.zeros(3, dtype=torch.int64)), "q_idx"),
    (dict(slots=torch.zeros(3, 4, dtype=i32)), "slots"),
    (dict(slots=torch.zeros(4, dtype=i32)), "slots"),
    (dict(rope=torch.zeros(8, 64)), "rope"),
    (dict(rope=torch.zeros(8, 2, 65)), "head_dim"),
    (dict(rope=torch.zeros(8, 2, 32, dtype=torch.float64)), "rope"),
    (dict(layout="pairs"), "layout"),
    (dict(seq_q=0), "seq_q"),
    (dict(block_size=0), "block_size"),
    (dict(V_scale=torch.ones(0)), "V_scale"),
    (dict(V_cache=torch.zeros(64, 128, dtype=torch.int16)), "V_cache"),
    (dict(K_cache=torch.zeros(63, 4, dtype=i32)), "K_cache"),
    (dict(Q_words=torch.zeros(3, 3, dtype=i32)), "Q_words"),
    (dict(slot_positions=torch.zeros(4, 31, dtype=i32)), "slot_positions"),
    (dict(block_tables=torch.zeros(4, 2, dtype=torch.int64)), "block_tables"),
    (dict(V_cache=torch.zeros(128, 64, dtype=torch.uint8).t()), "contiguous"),
    (dict(), "CUDA"),
])
def test_rope_cache_write_refuses(hyperion, change, match):
    with pytest.raises(RuntimeError, match=match):
        hyperion.rope_cache_write(**{**_write_args(), **change})


def _weights_args(n=4, group=2, seq_q=3, D=128, block=16, nb=2):
    return dict(Q=torch.zeros(n * group * seq_q, D // 32, dtype=i32), K_cache=torch.zeros(64, D // 32, dtype=i32),
                context_lens=torch.zeros(n, dtype=i32), block_tables=torch.zeros(n, nb, dtype=i32),
                weights=torch.zeros(n, nb * block), seq_q=seq_q, head_dim=D, block_size=block, num_blocks=nb,
                inv_sqrt_d=0.088, causal=False, kv_group=group)


@pytest.mark.parametrize("change, match", [
    (dict(head_dim=64), "head_dim"),
    (dict(context_lens=torch.zeros(4, dtype=torch.int64)), "context_lens"),
    (dict(kv_group=0), "kv_group"),
    (dict(n_q=0), "n_q"),
    (dict(seq_q=4), "Q smaller"),
    (dict(num_blocks=0), "num_blocks"),
    (dict(weights=torch.zeros(4, 31)), "weights"),
    (dict(weights=torch.zeros(4, 32, dtype=torch.float16)), "weights"),
    (dict(out=torch.zeros(4, 40)), "out"),
    (dict(q_first=torch.zeros(3, dtype=i32)), "q_first"),
    (dict(block_tables=torch.zeros(4, 1, dtype=i32)), "block_tables"),
    (dict(weights=torch.zeros(32, 4).t()), "contiguous"),
    (dict(), "CUDA"),
])
def test_accumulate_key_weights_refuses(hyperion, change, match):
    with pytest.raises(RuntimeError, match=match):
        hyperion.accumulate_key_weights(**{**_weights_args(), **change})


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan"), 1e39, -1e300])
@pytest.mark.parametrize("arg", ["inv_sqrt_d", "decay"])
def test_scales_that_are_not_finite_in_float32_are_refused(hyperion, arg, value):
    with pytest.raises(RuntimeError, match="finite"):
        hyperion.accumulate_key_weights(**{**_weights_args(), arg: value})


@pytest.mark.parametrize("cls, pack", [("RopeWriteArgs", "pack_rope_write"), ("KeyWeightsArgs", "pack_key_weights"),
                                       ("EvictArgs", "pack_evict")])
def test_packed_arguments_are_the_structures_bytes(hyperion, cls, pack):
    from hyperion_b200 import _capi
    args = getattr(_capi, cls)
    values = [0.37 + i if t is ctypes.c_float else 1 + i * 7 for i, (_, t) in enumerate(args._fields_)]
    back = args.from_buffer_copy(getattr(_capi, pack)(*values))
    for (name, t), v in zip(args._fields_, values):
        assert getattr(back, name) == (np.float32(v) if t is ctypes.c_float else v), name


def test_counts_beyond_int32_are_refused(hyperion):
    """Not cut to their low 32 bits: tensors without memory of their own stand for such counts."""
    n = (1 << 32) + 4
    x, ids = torch.zeros(1, 1, 128).expand(n, 1, 128), torch.zeros(1, dtype=i32).expand(n)
    with pytest.raises(RuntimeError, match="too many"):
        hyperion.rope_cache_write(**{**_write_args(), "Q_new": x, "K_new": x, "V_new": x, "seq_ids": ids, "positions": ids})
    heads = torch.zeros(1, 1, 128).expand(3, n, 128)
    with pytest.raises(RuntimeError, match="too many"):
        hyperion.rope_cache_write(**{**_write_args(), "K_new": heads, "V_new": heads})
    with pytest.raises(RuntimeError, match="too many"):
        hyperion.accumulate_key_weights(**{**_weights_args(), "context_lens": ids})
    with pytest.raises(RuntimeError, match="too many"):
        hyperion.evict_keys(**{**_evict_args(), "context_lens": ids})


def test_outputs_that_overlap_their_inputs_are_refused(hyperion):
    big = torch.zeros(9 * 32)
    with pytest.raises(RuntimeError, match="overlaps"):
        hyperion.accumulate_key_weights(**{**_weights_args(), "weights": big[:128].view(4, 32), "out": big[32:160].view(4, 32)})
    a = _evict_args()
    with pytest.raises(RuntimeError, match="overlaps"):
        hyperion.evict_keys(**{**a, "weights": big[:128].view(4, 32), "weights_out": big[4:132].view(4, 32)})
    pos = torch.zeros(9 * 32, dtype=i32)
    with pytest.raises(RuntimeError, match="overlaps"):
        hyperion.evict_keys(**{**a, "positions": pos[:128].view(4, 32), "positions_out": pos[4:132].view(4, 32)})
    ctx = torch.zeros(5, dtype=i32)
    with pytest.raises(RuntimeError, match="overlaps"):
        hyperion.evict_keys(**{**a, "context_lens": ctx[:4], "context_lens_out": ctx[1:]})


def _evict_args(n=4, D=128, block=16, nb=2):
    return dict(K_cache=torch.zeros(128, D // 32, dtype=i32), V_cache=torch.zeros(128, D, dtype=torch.uint8),
                context_lens=torch.zeros(n, dtype=i32), block_tables=None, block_size=block, num_blocks=nb,
                weights=torch.zeros(n, nb * block), positions=torch.zeros(n, nb * block, dtype=i32), keep=8)


@pytest.mark.parametrize("change, match", [
    (dict(V_cache=torch.zeros(128, 96, dtype=torch.uint8)), "V_cache"),
    (dict(V_cache=torch.zeros(128 * 128, dtype=torch.uint8)), "V_cache"),
    (dict(K_cache=torch.zeros(127, 4, dtype=i32)), "K_cache"),
    (dict(context_lens=torch.zeros(4)), "context_lens"),
    (dict(context_lens_out=torch.zeros(3, dtype=i32)), "context_lens_out"),
    (dict(weights=torch.zeros(4, 16)), "weights"),
    (dict(positions=torch.zeros(4, 32, dtype=torch.int64)), "positions"),
    (dict(positions=torch.zeros(4, 40, dtype=i32)), "positions"),
    (dict(weights_out=torch.zeros(4, 40)), "weights_out"),
    (dict(keep=-1), "keep"),
    (dict(keep=torch.zeros(4, dtype=torch.int64)), "keep"),
    (dict(keep=torch.zeros(3, dtype=i32)), "keep"),
    (dict(sink=-1), "sink"),
    (dict(recent=1 << 31), "recent"),
    (dict(V_scale=torch.ones(4)), "V_scale"),
    (dict(block_tables=torch.zeros(1, 2, dtype=i32)), "block_tables"),
    (dict(weights=torch.zeros(32, 4).t()), "contiguous"),
    (dict(), "CUDA"),
])
def test_evict_keys_refuses(hyperion, change, match):
    with pytest.raises(RuntimeError, match=match):
        hyperion.evict_keys(**{**_evict_args(), **change})


def _c(struct, **fields):
    a = struct()
    for k, v in fields.items():
        setattr(a, k, v)
    return a


FAKE = 4096  # an aligned address that no check reads


def test_c_boundary_refuses_rope_writes(hyperion):
    from hyperion_b200 import _capi

    good = dict(q=FAKE, k=FAKE, v=FAKE, in_dtype=1, n_tokens=2, n_heads=4, n_kv_heads=2, head_dim=128, rotary_dim=64,
                layout=0, n_positions=8, rope=FAKE, seq_ids=FAKE, positions=FAKE, seq_q=1, q_words=FAKE, q_rows=8,
                block_size=16, num_blocks=2, v_scale=FAKE, v_scale_numel=1, k_cache=FAKE, v_cache=FAKE, pool_rows=64)

    def call(ws=FAKE, nbytes=256, **change):
        a = _c(_capi.RopeWriteArgs, **{**good, **change})
        return _capi.lib.hyperion_rope_cache_write(ctypes.byref(a), ws, nbytes, None)

    INV, UNS, WSP = _capi.HYPERION_ERR_INVALID_ARG, _capi.HYPERION_ERR_UNSUPPORTED, _capi.HYPERION_ERR_WORKSPACE
    assert _capi.lib.hyperion_rope_cache_write(None, FAKE, 256, None) == INV
    for change, rc in [(dict(in_dtype=3), INV), (dict(head_dim=64), UNS), (dict(n_tokens=-1), INV), (dict(n_heads=0), INV),
                       (dict(rotary_dim=130), INV), (dict(rotary_dim=3), INV), (dict(layout=2), INV),
                       (dict(n_positions=0), INV), (dict(seq_q=0), INV), (dict(q_rows=-1), INV), (dict(v_scale_numel=0), INV),
                       (dict(block_size=0), INV), (dict(pool_rows=0), INV), (dict(block_tables_numel=4), INV),
                       (dict(block_size=1 << 20, num_blocks=1 << 12), UNS), (dict(q=None), INV), (dict(rope=None), INV),
                       (dict(q=FAKE + 1), INV), (dict(k_cache=FAKE + 4), INV), (dict(slot_rows=3), INV),
                       (dict(n_tokens=1 << 30), UNS), (dict(ws=None), WSP), (dict(nbytes=255), WSP), (dict(ws=FAKE + 16), WSP)]:
        assert call(**change) == rc, change
        assert _capi.last_error()
    assert call(n_tokens=0, q=None, rope=None) == _capi.HYPERION_OK


def test_c_boundary_refuses_key_weights(hyperion):
    from hyperion_b200 import _capi

    good = dict(q=FAKE, k_cache=FAKE, pool_rows=64, context_lens=FAKE, n_kv=2, kv_group=4, seq_q=128, n_q=100, head_dim=128,
                block_size=16, num_blocks=2, inv_sqrt_d=0.1, decay=1.0, weights=FAKE, weights_out=FAKE, weights_ld=32,
                scratch=FAKE, scratch_bytes=1 << 30)

    def call(ws=FAKE, nbytes=256, **change):
        a = _c(_capi.KeyWeightsArgs, **{**good, **change})
        return _capi.lib.hyperion_accumulate_key_weights(ctypes.byref(a), ws, nbytes, None)

    INV, UNS, WSP = _capi.HYPERION_ERR_INVALID_ARG, _capi.HYPERION_ERR_UNSUPPORTED, _capi.HYPERION_ERR_WORKSPACE
    assert _capi.lib.hyperion_accumulate_key_weights(None, FAKE, 256, None) == INV
    for change, rc in [(dict(head_dim=64), UNS), (dict(n_kv=-1), INV), (dict(kv_group=0), INV), (dict(seq_q=0), INV),
                       (dict(n_q=0), INV), (dict(inv_sqrt_d=math.nan), INV), (dict(decay=math.inf), INV),
                       (dict(block_tables=FAKE, block_tables_numel=3), INV), (dict(weights_ld=31), INV),
                       (dict(n_kv=1 << 24, weights_ld=32, kv_group=8), UNS), (dict(weights=None), INV), (dict(q=FAKE + 4), INV),
                       (dict(scratch=None), WSP), (dict(scratch_bytes=1), WSP), (dict(ws=None), WSP)]:
        assert call(**change) == rc, change
    assert call(n_kv=0, q=None) == _capi.HYPERION_OK


def test_c_boundary_refuses_evictions(hyperion):
    from hyperion_b200 import _capi

    good = dict(k_cache=FAKE, v_cache=FAKE, pool_rows=64, head_dim=128, n_kv=2, context_lens=FAKE, context_lens_out=FAKE,
                block_size=16, num_blocks=2, weights=FAKE, weights_out=FAKE, positions=FAKE, positions_out=FAKE, ld=32,
                keep=4, scratch=FAKE, scratch_bytes=1 << 30)

    def call(ws=FAKE, nbytes=256, **change):
        a = _c(_capi.EvictArgs, **{**good, **change})
        return _capi.lib.hyperion_evict_keys(ctypes.byref(a), ws, nbytes, None)

    INV, UNS, WSP = _capi.HYPERION_ERR_INVALID_ARG, _capi.HYPERION_ERR_UNSUPPORTED, _capi.HYPERION_ERR_WORKSPACE
    assert _capi.lib.hyperion_evict_keys(None, FAKE, 256, None) == INV
    for change, rc in [(dict(head_dim=96), UNS), (dict(n_kv=-1), INV), (dict(keep=-1), INV), (dict(sink=-1), INV),
                       (dict(recent=-1), INV), (dict(ld=31), INV), (dict(block_tables_numel=4), INV),
                       (dict(positions=None), INV), (dict(v_cache=FAKE + 8), INV), (dict(scratch=None), WSP),
                       (dict(scratch_bytes=3), WSP), (dict(ws=FAKE + 1), WSP)]:
        assert call(**change) == rc, change
    assert call(n_kv=0, weights=None) == _capi.HYPERION_OK


def test_rope_table_values_and_scaling():
    from hyperion_b200 import glue

    t = glue.rope_table(70000, 32, 500000.0).numpy()
    p, j = 69999, 3
    angle = p * 500000.0 ** (-2 * j / 32)
    assert t.shape == (70000, 2, 16) and t.dtype == np.float32
    assert t[p, 0, j] == np.float32(math.cos(angle)) and t[p, 1, j] == np.float32(math.sin(angle))
    # linear: position 4p of the scaled table is position p of the plain one (a quarter is exact)
    assert np.array_equal(glue.rope_table(41, 16, scaling="linear", factor=4.0).numpy()[::4],
                          glue.rope_table(11, 16).numpy())
    a, b = (np.arcsin(glue.rope_table(2, 16, **k).numpy()[1, 1].astype(np.float64)) for k in
            (dict(), dict(scaling="base", factor=8.0)))
    assert abs(b[0] - a[0]) < 1e-6 and abs(a[-1] / b[-1] - 8.0) < 0.05  # fastest kept, slowest slowed by the factor
    f = np.arcsin(glue.rope_table(2, 64, scaling="bands", factor=8.0, original_positions=4096).numpy()[1, 1].astype(np.float64))
    g = np.arcsin(glue.rope_table(2, 64).numpy()[1, 1].astype(np.float64))
    turns = 4096 * 10000.0 ** (-np.arange(0, 64, 2) / 64) / (2 * math.pi)
    assert np.allclose(f[turns > 32], g[turns > 32], rtol=1e-6) and np.allclose(f[turns < 1] * 8, g[turns < 1], rtol=1e-5)
    between = (turns > 1.1) & (turns < 31)
    assert np.all(f[between] < g[between]) and np.all(f[between] > g[between] / 8)


@pytest.mark.parametrize("bad", [dict(n_positions=0), dict(rotary_dim=7), dict(base=0.0), dict(factor=-1.0),
                                 dict(scaling="other"), dict(scaling="bands"), dict(scaling="base", rotary_dim=2)])
def test_rope_table_refuses(bad):
    from hyperion_b200 import glue

    with pytest.raises(ValueError):
        glue.rope_table(**{**dict(n_positions=4, rotary_dim=8), **bad})
