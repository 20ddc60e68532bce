"""Microscaled 4-bit format without a GPU: geometry, slot layout, checkpoints,
refusals of the C entry points, the oracle against the format's own rule."""

import ctypes
import json

import numpy as np
import pytest
import torch

from pagedmoe_amd import _lib, checkpoint as ck, kernels as K
from pagedmoe_amd.slab import component_specs
from tests import mx_oracle as M


@pytest.mark.parametrize("hidden,inter", [(32, 32), (96, 160), (4096, 1536), (8192, 8192)])
def test_geometry(hidden, inter):
    g = _lib.geom(hidden, inter, 4, 32)
    assert _lib.is_mx(g) and not _lib.is_mx(_lib.geom(64, 64, 4))
    half, scale = hidden * inter // 2, hidden * inter // 32
    assert list(g.nbytes) == [half, scale, 0] * 3
    assert all(o % 256 == 0 for o in g.off) and g.expert_bytes % 256 == 0
    ends = [g.off[c] + g.nbytes[c] for c in range(9)]
    assert all(ends[c] <= g.off[c + 1] for c in range(8)) and ends[8] <= g.expert_bytes
    specs = component_specs(g)
    assert list(specs) == [f"{p}_proj.{c}" for p in ("gate", "up", "down")
                           for c in ("weight", "scales")]
    assert specs["down_proj.scales"] == ((hidden, inter // 32), torch.uint8, scale, g.off[7])


@pytest.mark.parametrize("args", [(96, 96, 6, 32), (100, 96, 4, 32), (96, 0, 4, 32),
                                  (128, 128, 4, 16), (96, 128, 4, 64)])
def test_geometry_refusals(args):
    with pytest.raises(_lib.PmoeError):
        _lib.geom(*args)


def test_group_forms_of_the_other_format_stay_off():
    g = _lib.geom(1024, 512, 4, 32)
    L = _lib.lib()
    for n in (1, 20, 100, 3000):
        assert L.pmoe_stream_wanted(ctypes.byref(g), n, 4, 32, 0) == 0
        assert L.pmoe_prefill_wide(ctypes.byref(g), None, None, n, 4, 32) == 0


D = ctypes.c_void_p(0x1000)


@pytest.mark.parametrize("w,dtype,rows,cols,q,s,msg", [
    (None, 0, 4, 32, D, D, b"null"), (D, 0, 4, 32, None, D, b"null"), (D, 0, 4, 32, D, None, b"null"),
    (D, 3, 4, 32, D, D, b"dtype"), (D, -1, 4, 32, D, D, b"dtype"), (D, 0, 4, 48, D, D, b"multiple"),
    (D, 0, 4, 0, D, D, b"multiple"), (D, 0, -1, 32, D, D, b"multiple"),
    (ctypes.c_void_p(0x1001), 1, 4, 32, D, D, b"misaligned"),
    (D, 1, 4, 32, ctypes.c_void_p(0x1002), D, b"misaligned")])
def test_format_refusals(w, dtype, rows, cols, q, s, msg):
    """Refused on the host, nothing is launched, the dummy pointers never read."""
    L = _lib.lib()
    assert L.pmoe_mx4_quantize(w, dtype, rows, cols, q, s, None) == -1
    assert msg in L.pmoe_last_error()
    assert L.pmoe_mx4_dequant(q, s, rows, cols, dtype, w, None) == -1
    assert msg in L.pmoe_last_error()


def test_format_of_no_rows_launches_nothing():
    L = _lib.lib()
    assert L.pmoe_mx4_quantize(D, 0, 0, 32, D, D, None) == 0
    assert L.pmoe_mx4_dequant(D, D, 0, 32, 2, D, None) == 0


def test_wrappers_refuse_host_tensors():
    with pytest.raises(ValueError):
        K.mx4_quantize(torch.zeros(2, 32))
    with pytest.raises(TypeError):
        K.mx4_quantize(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(ValueError):
        K.mx4_dequant(torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 1, dtype=torch.uint8))


@pytest.mark.parametrize("change", ["group", "bits", "dims", "big", "slot", "off", "slab"])
def test_expert_entries_refuse_bad_geometries(change):
    L = _lib.lib()
    g = _lib.geom(1024, 512, 4, 32)
    slab = 0x1000
    if change == "group":
        g.group = 16
    elif change == "bits":
        g.bits = 6
    elif change == "dims":
        g.inter = 500
    elif change == "big":
        g.hidden = 8224
    elif change == "slot":
        g.expert_bytes += 8
    elif change == "off":
        g.off[6] += 4
    else:
        slab += 8
    p = ctypes.byref(g)
    s = ctypes.c_void_p(slab)
    rc = _lib.RouteCfg()
    rc.n_experts, rc.top_k, rc.routed_scale = 8, 2, 1.0
    assert L.pmoe_switch_glu(p, s, D, 8, D, D, 1, 2, D, D, 1 << 40, None) == -1
    assert b"geometry" in L.pmoe_last_error()
    assert L.pmoe_moe_experts(p, s, D, 8, D, D, D, 1, 2, -1, None, D, D, 1 << 40, None) == -1
    assert L.pmoe_moe_block(p, ctypes.byref(rc), s, D, D, None, None, D, 1, -1, None, D, D, D, D,
                            1 << 40, None) == -1


@pytest.mark.parametrize("which", ["x", "out"])
def test_expert_entries_refuse_rows_off_16_bytes(which):
    L = _lib.lib()
    g = _lib.geom(1024, 512, 4, 32)
    p = ctypes.byref(g)
    x, out = (ctypes.c_void_p(0x1002 if which == n else 0x1000) for n in ("x", "out"))
    rc = _lib.RouteCfg()
    rc.n_experts, rc.top_k, rc.routed_scale = 8, 2, 1.0
    assert L.pmoe_switch_glu(p, D, D, 8, x, D, 1, 2, out, D, 1 << 40, None) == -1
    assert b"16 bytes" in L.pmoe_last_error()
    assert L.pmoe_moe_experts(p, D, D, 8, x, D, D, 1, 2, -1, None, out, D, 1 << 40, None) == -1
    assert L.pmoe_moe_block(p, ctypes.byref(rc), D, D, D, None, None, x, 1, -1, None, out, D, D, D,
                            1 << 40, None) == -1
    assert b"16 bytes" in L.pmoe_last_error()


@pytest.mark.parametrize("hidden,inter,k,shared,experts", [
    (32, 32, 1, 0, 1), (1024, 512, 4, 0, 32), (2048, 512, 10, 1, 512), (4096, 1536, 8, 0, 128),
    (7168, 2048, 8, 1, 384), (32, 8192, 64, 0, 64), (64, 8192, 2, 1, 1000)])
def test_workspace_of_a_call_serves_shorter_ones(hidden, inter, k, shared, experts):
    L = _lib.lib()
    g = _lib.geom(hidden, inter, 4, 32)
    need = [L.pmoe_moe_workspace(ctypes.byref(g), n, k, shared, experts) for n in range(1, 80)]
    assert need == sorted(need)


def test_expert_entries_refuse_a_small_workspace():
    L = _lib.lib()
    g = _lib.geom(1024, 512, 4, 32)
    need = L.pmoe_moe_workspace(ctypes.byref(g), 5, 2, 0, 8)
    assert L.pmoe_switch_glu(ctypes.byref(g), D, D, 8, D, D, 5, 2, D, D, need - 1, None) == -5


@pytest.mark.parametrize("hidden,inter,n,k", [
    (1024, 512, 1 << 24, 1),     # the split's blocks
    (8192, 512, 1 << 22, 2),     # the combine's
    (1056, 480, 3 << 20, 4),     # small tiles
    (8192, 8192, 700000, 8)])    # large ones
def test_expert_entries_refuse_more_rows_than_a_launch_holds(hidden, inter, n, k):
    """On the host, before the first launch; the dummy pointers are never read."""
    L = _lib.lib()
    p = ctypes.byref(_lib.geom(hidden, inter, 4, 32))
    assert L.pmoe_switch_glu(p, D, D, 8, D, D, n, k, D, D, 1 << 60, None) == -1
    assert b"too many rows" in L.pmoe_last_error()
    assert L.pmoe_moe_experts(p, D, D, 8, D, D, D, n, k, -1, None, D, D, 1 << 60, None) == -1
    assert b"too many rows" in L.pmoe_last_error()


# ---------------------------------------------------------------- the oracle

def test_oracle_rounds_to_nearest_with_ties_to_even():
    # a group whose largest is 7.5 (scale 1): every midpoint, both signs
    mids = (M.E2M1[1:] + M.E2M1[:-1]) / 2
    w = np.zeros((1, 32))
    w[0, :7], w[0, 7:14], w[0, 14] = mids, -mids, 7.5
    codes, scales = M.quantize(w)
    assert scales[0, 0] == 127
    even = [0, 2, 2, 4, 4, 6, 6]
    assert codes[0, :7].tolist() == even and codes[0, 7:14].tolist() == [c | 8 for c in even]
    assert codes[0, 14] == 7
    assert np.array_equal(M.unpack(M.pack(codes)), codes)


@pytest.mark.parametrize("top,scale", [(1.0, 125), (3.99, 126), (4.0, 127), (2.0 ** -126, 0),
                                       (2.0 ** -149, 0), (2.0 ** 127, 252), (0.0, 0)])
def test_oracle_scales(top, scale):
    w = np.zeros((1, 32))
    w[0, 5] = -top
    assert M.quantize(w)[1][0, 0] == scale


# ---------------------------------------------------------------- checkpoints

def write_safetensors(path, tensors):
    head, at = {}, 0
    for name, a in tensors.items():
        dt = {"uint32": "U32", "uint8": "U8", "uint16": "BF16"}[a.dtype.name]
        head[name] = {"dtype": dt, "shape": list(a.shape), "data_offsets": [at, at + a.nbytes]}
        at += a.nbytes
    blob = json.dumps(head).encode()
    with open(path, "wb") as f:
        f.write(len(blob).to_bytes(8, "little") + blob)
        for a in tensors.values():
            f.write(np.ascontiguousarray(a).tobytes())


def make_checkpoint(path, hidden, inter, experts, layers=1, stacked=True, biases=False,
                    scale_dtype=np.uint8):
    rng = np.random.default_rng(0)
    tensors = {}
    for li in range(layers):
        for proj, rows, cols in (("gate_proj", inter, hidden), ("up_proj", inter, hidden),
                                 ("down_proj", hidden, inter)):
            w = rng.integers(0, 1 << 32, (experts, rows, cols // 8), dtype=np.uint32)
            s = rng.integers(110, 130, (experts, rows, cols // 32)).astype(scale_dtype)
            comps = {"weight": w, "scales": s}
            if biases:
                comps["biases"] = s
            for comp, a in comps.items():
                if stacked:
                    tensors[f"model.layers.{li}.mlp.switch_mlp.{proj}.{comp}"] = a
                else:
                    for e in range(experts):
                        tensors[f"model.layers.{li}.mlp.experts.{e}.{proj}.{comp}"] = a[e]
    write_safetensors(path / "model.safetensors", tensors)
    return tensors


@pytest.mark.parametrize("stacked", [True, False])
def test_checkpoint_bytes_land_in_the_slot(tmp_path, stacked):
    hidden, inter, experts = 96, 64, 3
    t = make_checkpoint(tmp_path, hidden, inter, experts, stacked=stacked)
    index = ck.read_headers(tmp_path)
    (_, path), = ck.find_moe_layers(index)
    lay = ck.layer_layout(path, index)
    assert lay.microscaled and lay.geometry(32) == (hidden, inter, 4)
    g = _lib.geom(hidden, inter, 4, 32)
    ck.check_layout(lay, g)
    specs = component_specs(g)
    for e in range(experts):
        out = np.zeros(int(g.expert_bytes), np.uint8)
        ck.read_expert(lay, e, g, out)
        for name, (shape, _, nb, off) in specs.items():
            src = (t[f"{path}.{name}"][e] if stacked else
                   t[f"{path.rsplit('.', 1)[0]}.experts.{e}.{name}"])
            assert out[off:off + nb].tobytes() == src.tobytes(), (e, name)


def test_checkpoint_of_another_format_is_refused(tmp_path):
    """bf16 scales without biases are no format; a microscaled layout does not
    fit an affine slot, nor an affine one a microscaled slot."""
    a, b, c = (tmp_path / n for n in "abc")
    for p in (a, b, c):
        p.mkdir()
    make_checkpoint(a, 64, 64, 2, scale_dtype=np.uint16)
    index = ck.read_headers(a)
    with pytest.raises(KeyError):
        ck.layer_layout("model.layers.0.mlp.switch_mlp", index)
    make_checkpoint(b, 64, 64, 2)
    lay = ck.layer_layout("model.layers.0.mlp.switch_mlp", ck.read_headers(b))
    with pytest.raises((_lib.PmoeError, KeyError)):
        ck.check_layout(lay, _lib.geom(64, 64, 4, 64))
    make_checkpoint(c, 64, 64, 2, biases=True, scale_dtype=np.uint16)
    lay = ck.layer_layout("model.layers.0.mlp.switch_mlp", ck.read_headers(c))
    with pytest.raises(_lib.PmoeError):
        ck.check_layout(lay, _lib.geom(64, 64, 4, 32))
