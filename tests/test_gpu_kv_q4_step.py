"""Whole decode steps over the 4-bit KV cache (tune model_kv_q4 at creation) against the CPU step whose caches hold the same values."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import cases
import q4_cache as host
import step_oracle as so
from test_gpu_decode_step import MINI_LLAMA, MINI_QWEN, cosine

pytestmark = pytest.mark.gpu


def create(ck, cfg, batch):
    so.bind_model_api(ck)
    ck.ckb200_tune_set(b"model_kv_q4", 1)
    try:
        return ck.ckb200_model_create(C.byref(so.make_cfg(cfg, batch=batch)))
    finally:
        ck.ckb200_tune_set(b"model_kv_q4", 0)


def as_pages(cache, rows):
    """fp32 [Hkv][tokens][d] -> the bytes of a page of `rows` rows."""
    out = np.zeros((cache.shape[0], rows, cache.shape[2] // 32 * host.BLOCK), dtype=np.uint8)
    out[:, :cache.shape[1]] = host.quantize(cache)
    return out


@pytest.mark.parametrize("graph", [0, 1], ids=["launches", "graph"])
@pytest.mark.parametrize("cfg,batch", [(MINI_QWEN, 1), (MINI_LLAMA, 2)])
def test_decode_steps_with_4_bit_cache(ck, orc, monkeypatch, cfg, batch, graph):
    cpu = so.CpuModel(cfg, seed=23)
    start = 33
    cpu.prefill_kv(start, seed=24)
    store = cases.kv_cache_store

    def store_4_bits(lib, prefix, kc, vc, k, v, pos):
        store(lib, prefix, kc, vc, k, v, pos)
        for c in (kc, vc):
            c[:, pos] = host.values(host.quantize(c[:, pos]), np.float32)

    monkeypatch.setattr(cases, "kv_cache_store", store_4_bits)
    ck.ckb200_tune_set(b"model_graph", graph)
    handle = create(ck, cfg, batch)
    assert handle, ck.ckb200_last_error_message()
    try:
        assert ck.ckb200_model_kv_element_bytes(handle) == 1
        caches, cpu.kc, cpu.vc = (cpu.kc, cpu.vc), np.zeros((len(cpu.layers), 0), np.float32), np.zeros((len(cpu.layers), 0), np.float32)
        so.upload_whole_model(ck, handle, cpu, batch)                    # the caches go up by themselves
        V, Hkv, d, S = cfg["vocab_size"], cfg["num_kv_heads"], cfg["head_dim"], cfg["max_seq_len"]
        rows = (S + 15) // 16 * 16
        for l in range(len(cpu.layers)):
            for is_v, c in enumerate(caches):
                page = as_pages(c[l, :, :start], rows)
                for b in range(batch):
                    assert ck.ckb200_copy_to_device(C.c_void_p(ck.ckb200_model_kv_device(handle, l, is_v) + b * page.nbytes), cases.vptr(page), page.nbytes) == 0
                c[l, :, :start] = host.values(host.quantize(c[l, :, :start]), np.float32)
        cpu.kc, cpu.vc = caches
        assert ck.ckb200_model_set_pos(handle, start) == 0
        for step, tok in enumerate([9, 41, 300]):
            want = cpu.decode(orc, tok, start + step)
            ids, logits = np.full(batch, tok, dtype=np.int32), np.full((batch, V), np.nan, dtype=np.float32)
            assert ck.ckb200_model_decode(handle, cases.vptr(ids), cases.vptr(logits)) == 0, ck.ckb200_last_error_message()
            for b in range(batch):
                assert cosine(logits[b], want) >= 0.9999, (step, b)
                assert float(np.max(np.abs(logits[b] - want))) / float(np.max(np.abs(want))) < 5e-3, (step, b)
        # layer 0's rows do not depend on earlier attention: the old ones are untouched, the new ones the CPU step's within a step of a code, the rest still zero
        got = np.zeros((batch, Hkv, rows, d // 32 * host.BLOCK), np.uint8)
        assert ck.ckb200_copy_to_host(cases.vptr(got), C.c_void_p(ck.ckb200_model_kv_device(handle, 0, 1)), got.nbytes) == 0
        for b in range(batch):
            values = host.values(got[b], np.float32)
            assert np.array_equal(values[:, :start], cpu.vc[0][:, :start])
            a, w = values[:, start:start + 3], cpu.vc[0][:, start:start + 3]
            spread = np.ptp(w.reshape(Hkv, 3, -1, 32), axis=-1).repeat(32, -1).reshape(w.shape)
            assert (np.abs(a - w) <= spread / 14).all()
            assert not got[b][:, start + 3:].any()
        assert ck.ckb200_model_reset(handle) == 0
    finally:
        ck.ckb200_tune_set(b"model_graph", 1)
        ck.ckb200_model_free(handle)


def test_prompts_and_synthetic_caches(ck):
    """A prompt runs as decode steps and leaves the logits that they leave; a synthetic cache is followed by steps with finite logits; an unsupported head size is refused."""
    handle = create(ck, MINI_QWEN, 1)
    assert handle, ck.ckb200_last_error_message()
    try:
        assert ck.ckb200_model_fill_synthetic(handle, 3) == 0
        V = MINI_QWEN["vocab_size"]
        ids, a, b = np.arange(1, 21, dtype=np.int32), np.zeros(V, np.float32), np.zeros(V, np.float32)
        assert ck.ckb200_model_prefill(handle, cases.vptr(ids), 20, cases.vptr(a)) == 0
        assert ck.ckb200_model_reset(handle) == 0
        for t in ids:
            one = np.array([t], dtype=np.int32)
            assert ck.ckb200_model_decode(handle, cases.vptr(one), cases.vptr(b)) == 0
        assert np.isfinite(a).all() and np.array_equal(a, b)
        assert ck.ckb200_model_fill_kv_synthetic(handle, 20, 4) == 0 and ck.ckb200_model_get_pos(handle) == 20
        assert ck.ckb200_model_decode(handle, cases.vptr(ids[:1].copy()), cases.vptr(b)) == 0
        assert np.isfinite(b).all() and not np.array_equal(a, b)
    finally:
        ck.ckb200_model_free(handle)
    assert not create(ck, dict(MINI_QWEN, head_dim=32, num_heads=12, num_kv_heads=4), 1)
    assert b"4-bit cache" in ck.ckb200_last_error_message()
    ck.ckb200_clear_error()
