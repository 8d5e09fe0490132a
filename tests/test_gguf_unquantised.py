"""Checkpoints whose routed experts are F16 or BF16: their geometry, and their
records in an arena, where the operators on grouped rows read them in place."""
import ctypes as C

import numpy as np
import pytest

H, I, E, USED, LAYERS = 128, 96, 5, 2, 2


def write(path, kind):
    """The file, and its experts as [layer][role] -> 16-bit words [E, rows, columns]."""
    from gguf import GGMLQuantizationType, GGUFWriter
    rng = np.random.default_rng(3)
    w = GGUFWriter(str(path), "qwen3moe")
    w.add_block_count(LAYERS)
    w.add_expert_count(E)
    w.add_expert_used_count(USED)
    words = []
    for L in range(LAYERS):
        words.append({})
        for role, rows, cols in (("down", H, I), ("gate", I, H), ("up", I, H)):
            v = (rng.standard_normal((E, rows, cols)) * 0.1).astype(np.float32)
            bits = v.astype(np.float16).view(np.uint16) if kind == "F16" else (v.view(np.uint32) >> 16).astype(np.uint16)
            words[L][role] = bits
            w.add_tensor(f"blk.{L}.ffn_{role}_exps.weight", bits.view(np.uint8), raw_dtype=GGMLQuantizationType[kind])
    w.write_header_to_file()
    w.write_kv_data_to_file()
    w.write_tensors_to_file()
    w.close()
    return words


@pytest.mark.parametrize("kind", ["F16", "BF16"])
def test_geometry(gxlib, tmp_path, kind):
    from galactus_b200 import _lib as L
    write(tmp_path / "m.gguf", kind)
    info = L.gx_gguf_moe()
    L.check(gxlib.lib().gx_gguf_moe_info(str(tmp_path / "m.gguf").encode(), C.byref(info)))
    t = {"F16": L.TYPE_F16, "BF16": L.TYPE_BF16}[kind]
    assert (info.type_down, info.type_gate, info.type_up, info.hidden, info.intermediate, info.experts) == (t, t, t, H, I, E)
    assert info.record_bytes_raw == 3 * H * I * 2 and info.record_bytes % 16384 == 0 and info.record_bytes >= info.record_bytes_raw


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["F16", "BF16"])
def test_products_on_the_loaded_records(gxlib, dev, tmp_path, kind):
    import torch
    from galactus_b200 import _lib as L
    from galactus_b200.models import ModelShape
    words = write(tmp_path / "m.gguf", kind)
    t, dtype = {"F16": (L.TYPE_F16, torch.float16), "BF16": (L.TYPE_BF16, torch.bfloat16)}[kind]
    m = ModelShape("unquantised", LAYERS, H, E, USED, I, t, t, t)
    arena = gxlib.Arena(m, capacity_bytes=LAYERS * E * m.record, policy=gxlib.POLICY_AUTO, max_tokens=8)
    try:
        n = C.c_uint32()
        gxlib.check(gxlib.lib().gx_arena_load_gguf(arena.h, str(tmp_path / "m.gguf").encode(), C.byref(n)), "gx_arena_load_gguf")
        assert n.value == E * LAYERS
        stream = torch.cuda.current_stream()
        arena.warm_all(stream)
        for layer in range(LAYERS):
            base, record, slots = arena.layer_view(layer)
            order = [e for e in range(E)]
            at = [arena.slot_of(layer, e) for e in order]
            offsets = np.zeros(slots + 1, np.int32)
            for s in at:
                offsets[s + 1:] += 1                                  # one row for every loaded slot
            rows = sorted(range(E), key=lambda e: at[e])
            x = torch.randn((E, I), device="cuda").to(dtype)
            y = torch.empty((E, H), device="cuda")
            off = torch.from_numpy(offsets).cuda()
            gxlib.check(gxlib.lib().gx_mul_mat_grouped(t, base, I, H, 2 * I, record, slots, x.data_ptr(), E, 2 * I, off.data_ptr(),
                                                       None, E, 0, 0, L.TYPE_F32, y.data_ptr(), 4 * H, stream.cuda_stream))
            for j, e in enumerate(rows):
                wt = torch.from_numpy(words[layer]["down"][e].view(np.int16)).cuda().view(dtype).double()
                want = wt @ x[j].double()
                tol = (wt.abs() @ x[j].double().abs()) * (I / 16 + 16) * 2.0 ** -23 + 2.0 ** -24 * want.abs()
                assert bool(((y[j].double() - want).abs() <= tol).all())
    finally:
        arena.close()
