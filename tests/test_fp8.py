"""Block-scaled FP8: what needs no GPU - C ABI refusals, fake kernels, the layer's loaders and the config's routing."""

import pytest
import torch
from torch import nn

from fp8_util import half_step, near
from sglang_exl3 import _lib, ops
from sglang_exl3.exl3 import EXL3Config, EXL3LinearMethod
from sglang_exl3.fp8 import FP8BlockLinearMethod, fp8_block_modules, is_fp8_block_config

P = 1 << 12  # an aligned address that is never read


@pytest.fixture(scope="module", autouse=True)
def _registered():
    ops.register_custom_ops()


def test_oracle_rounding():
    """The oracle's e4m3 rounding against torch's conversion, at every value and between neighbours."""
    bits = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double()
    v = bits[bits.isfinite()].sort().values
    mid = (v[1:] + v[:-1]) / 2
    for t in (v, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)):
        assert torch.equal(near(t), t.float().to(torch.float8_e4m3fn).double())
        assert bool(((near(t) - t).abs() <= half_step(t)).all())


@pytest.mark.parametrize("call,text", [
    (("exl3_fp8_quant_rows", P, 128, P, P, 2, 1, 128, None), b"dtype=2"),
    (("exl3_fp8_quant_rows", P, 128, P, P, 1, 1, 120, None), b"cols=120"),
    (("exl3_fp8_quant_rows", P, 128, P, P, 1, -1, 128, None), b"rows=-1"),
    (("exl3_fp8_quant_rows", P, 128, P, P, 1, 0x7fffffff, 256, None), b"too large"),
    (("exl3_fp8_quant_rows", None, 128, P, P, 1, 1, 128, None), b"null pointer"),
    (("exl3_fp8_quant_rows", P + 2, 128, P, P, 1, 1, 128, None), b"16-byte aligned"),
    (("exl3_fp8_quant_rows", P, 124, P, P, 1, 1, 128, None), b"row stride"),
    (("exl3_fp8_quant_rows", P, 132, P, P, 1, 2, 128, None), b"row stride"),
    (("exl3_fp8_quant_rows", P, 128, P + 4, P, 1, 1, 128, None), b"misaligned"),
    (("exl3_fp8_norm_quant", P, 128, None, 0, None, 1e-6, None, None, P, P, 1, 1, 128, None), b"null pointer"),
    (("exl3_fp8_norm_quant", P, 128, None, 0, P, 1e-6, P, None, P, P, 1, 1, 128, None), b"null pointer"),
    (("exl3_fp8_norm_quant", P, 128, None, 0, P, -1.0, None, None, P, P, 1, 1, 128, None), b"eps"),
    (("exl3_fp8_norm_quant", P, 128, None, 0, P, float("nan"), None, None, P, P, 1, 1, 128, None), b"eps"),
    (("exl3_fp8_norm_quant", P, 32784, None, 0, P, 1e-6, None, None, P, P, 1, 1, 32784, None), b"above 32768"),
    (("exl3_fp8_norm_quant", P, 128, P, 64, P, 1e-6, P, None, P, P, 1, 1, 128, None), b"row strides"),
    (("exl3_fp8_norm_quant", P, 128, None, 0, P + 2, 1e-6, None, None, P, P, 1, 1, 128, None), b"misaligned"),
    (("exl3_fp8_swiglu_quant", P, 256, -1.0, P, P, 1, 1, 128, None), b"limit"),
    (("exl3_fp8_swiglu_quant", P, 256, float("nan"), P, P, 1, 1, 128, None), b"limit"),
    (("exl3_fp8_swiglu_quant", P, 248, 0.0, P, P, 1, 1, 128, None), b"row stride"),
    (("exl3_fp8_linear", P, 3, P, P, P, None, P, 1, 1, 120, 128, None, 0, None), b"k=120"),
    (("exl3_fp8_linear", P, 3, P, P, P, None, P, 1, -1, 128, 128, None, 0, None), b"m=-1"),
    (("exl3_fp8_linear", P, 2, P, P, P, None, P, 1, 1, 128, 128, None, 0, None), b"x dtype=2"),
    (("exl3_fp8_linear", P, 3, P, P, P, None, P, 2, 1, 128, 128, None, 0, None), b"y dtype=2"),
    (("exl3_fp8_linear", P, 3, None, P, P, None, P, 1, 1, 128, 128, None, 0, None), b"null pointer"),
    (("exl3_fp8_linear", P, 3, P, P + 8, P, None, P, 1, 1, 128, 128, None, 0, None), b"misaligned"),
])
def test_abi_refuses_before_the_device(call, text):
    L = _lib.lib()
    assert getattr(L, call[0])(*call[1:]) == _lib.EXL3_ERR_ARG
    assert text in L.exl3_last_error()


def test_abi_workspace_and_empty_calls():
    L = _lib.lib()
    need = L.exl3_fp8_linear_workspace_size(_lib.DTYPE_BF16, 5, 400, 64)
    assert need >= 5 * 400 + 5 * 4 * 4
    rc = L.exl3_fp8_linear(P, 1, None, P, P, None, P, 1, 5, 400, 64, P, need - 1, None)
    assert rc == _lib.EXL3_ERR_WORKSPACE
    assert L.exl3_fp8_linear_workspace_size(_lib.DTYPE_BF16, 0, 400, 64) == 0
    assert L.exl3_fp8_linear_workspace_size(_lib.DTYPE_BF16, 5, 401, 64) == 0
    assert L.exl3_fp8_linear(None, 1, None, None, None, None, None, 1, 0, 400, 64, None, 0, None) == _lib.EXL3_OK
    assert L.exl3_fp8_quant_rows(None, 128, None, None, 1, 0, 128, None) == _lib.EXL3_OK


def test_fake_kernels_and_cpu_refusal():
    from torch._subclasses.fake_tensor import FakeTensorMode

    o = torch.ops.sglang_exl3
    with FakeTensorMode():
        x = torch.empty((2, 3, 272), dtype=torch.bfloat16)
        w, ws = torch.empty((200, 272), dtype=torch.float8_e4m3fn), torch.empty((2, 3))
        q, s = o.fp8_quant_rows(x)
        assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and s.shape == (2, 3, 3)
        out = o.fp8_norm_quant(x, torch.empty(272, dtype=torch.bfloat16), 1e-6, x, True)
        assert [tuple(t.shape) for t in out] == [(2, 3, 272), (2, 3, 3), (2, 3, 272), (2, 3, 272)]
        assert len(o.fp8_norm_quant(x, torch.empty(272, dtype=torch.bfloat16), 1e-6)) == 2
        q2, s2 = o.fp8_swiglu_quant(torch.empty((4, 544), dtype=torch.float16), 1.0)
        assert q2.shape == (4, 272) and s2.shape == (4, 3)
        y = o.fp8_linear(q, w, ws, s, None, False)
        assert y.shape == (6, 200) and y.dtype == torch.float16
    for call in (lambda: o.fp8_quant_rows(torch.zeros((1, 128)).bfloat16()),
                 lambda: o.fp8_swiglu_quant(torch.zeros((1, 256)).bfloat16()),
                 lambda: o.fp8_norm_quant(torch.zeros((1, 128)).bfloat16(), torch.ones(128).bfloat16(), 1e-6),
                 lambda: o.fp8_linear(torch.zeros((1, 128)).bfloat16(), torch.zeros((1, 128)).to(torch.float8_e4m3fn),
                                      torch.ones((1, 1)))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


# --------------------------------------------------------------------- the layer

def _layer(k, widths, dtype=torch.bfloat16):
    layer, method = nn.Module(), FP8BlockLinearMethod()
    method.create_weights(layer, k, widths, k, sum(widths), dtype)
    return layer, method


def _e4m3(n, k):
    return torch.randint(0, 120, (n, k), dtype=torch.uint8).view(torch.float8_e4m3fn)


def _u8(t):
    return t.view(torch.uint8)


def test_layer_shards_land_in_their_rows():
    layer, method = _layer(272, [256, 128, 72])
    assert layer.weight.shape == (456, 272) and layer.weight_scale_inv.shape == (4, 3)
    parts = [(_e4m3(n, 272), torch.rand((-(-n // 128), 3))) for n in (256, 128, 72)]
    with pytest.raises(RuntimeError, match="received no"):
        method.process_weights_after_loading(layer)
    for i, (w, s) in enumerate(parts):
        layer.weight.weight_loader(layer.weight, w, i if i else "q")
        layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, s, "qkv"[i])
    method.process_weights_after_loading(layer)
    assert torch.equal(_u8(layer.weight.data), _u8(torch.cat([w for w, _ in parts])))
    assert torch.equal(layer.weight_scale_inv.data, torch.cat([s for _, s in parts]))
    # the same, stored as one tensor
    other, method = _layer(272, [256, 128, 72])
    other.weight.weight_loader(other.weight, layer.weight.data.clone())
    other.weight_scale_inv.weight_loader(other.weight_scale_inv, layer.weight_scale_inv.data.clone())
    method.process_weights_after_loading(other)
    assert torch.equal(_u8(other.weight.data), _u8(layer.weight.data))


def test_layer_parts_of_a_rank(monkeypatch):
    """Each rank of two takes its half of the rows or of the columns, in whole blocks."""
    from sglang_exl3 import exl3

    w, s = _e4m3(512, 768), torch.rand((4, 6))
    for rank in (0, 1):
        monkeypatch.setattr(exl3, "_tp_rank_size", lambda: (rank, 2))
        layer, _ = _layer(768, [256])
        layer.weight.weight_loader(layer.weight, w)
        layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, s)
        assert torch.equal(_u8(layer.weight.data), _u8(w)[256 * rank:256 * rank + 256])
        assert torch.equal(layer.weight_scale_inv.data, s[2 * rank:2 * rank + 2])
        layer, _ = _layer(384, [512])
        layer.weight.weight_loader(layer.weight, w)
        layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, s)
        assert torch.equal(_u8(layer.weight.data), _u8(w)[:, 384 * rank:384 * rank + 384])
        assert torch.equal(layer.weight_scale_inv.data, s[:, 3 * rank:3 * rank + 3])
    layer, _ = _layer(768, [64])  # half of one block of scales
    with pytest.raises(ValueError, match="whole blocks"):
        layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, torch.rand((2, 6)))


def test_layer_refuses():
    with pytest.raises(ValueError, match="multiple of 16"):
        _layer(200, [128])
    with pytest.raises(ValueError, match="inside a block"):
        _layer(256, [64, 128])
    layer, method = _layer(256, [128, 128])
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        layer.weight.weight_loader(layer.weight, torch.zeros((128, 256), dtype=torch.bfloat16), 0)
    with pytest.raises(ValueError, match="shard"):
        layer.weight.weight_loader(layer.weight, _e4m3(128, 256), 2)
    with pytest.raises(ValueError, match="shape"):
        layer.weight.weight_loader(layer.weight, _e4m3(128, 128), 1)
    with pytest.raises(ValueError, match="rows"):
        layer.weight.weight_loader(layer.weight, _e4m3(128, 256))


# -------------------------------------------------------------------- the config

class RowParallelLinear(nn.Module):
    pass


class ParallelLMHead(nn.Module):
    pass


FP8 = {"quant_method": "fp8", "fmt": "e4m3", "weight_block_size": [128, 128], "activation_scheme": "dynamic",
       "modules_to_not_convert": ["model.layers.3", "shared_head"]}


def _method(cfg, prefix, layer=None):
    return cfg.get_quant_method(layer or RowParallelLinear(), prefix)


def test_routing_by_quantization(monkeypatch):
    def config(q, **more):
        return EXL3Config.from_config({"quant_method": "exl3", "bits": 3, "scope": "glm53_routed_experts_only",
                                       "non_routed_quantization": q, **more})

    cfg = config(FP8)
    assert isinstance(_method(cfg, "model.layers.0.self_attn.o_proj"), FP8BlockLinearMethod)
    for left_out in ("model.layers.3.self_attn.o_proj", "model.layers.9.shared_head", "mtp.layers.0.o_proj"):
        assert not isinstance(_method(cfg, left_out), FP8BlockLinearMethod)
    assert isinstance(_method(cfg, "model.layers.30.self_attn.o_proj"), FP8BlockLinearMethod)
    assert not isinstance(_method(cfg, "lm_head", ParallelLMHead()), FP8BlockLinearMethod)
    for q in (None, "fp8", {"quant_method": "fp8"}, {**FP8, "weight_block_size": [1, 128]},
              {**FP8, "activation_scheme": "static"}, {**FP8, "fmt": "e5m2"}, {**FP8, "quant_method": "int8"}):
        assert not is_fp8_block_config(q)
        assert not isinstance(_method(config(q), "model.layers.0.self_attn.o_proj"), FP8BlockLinearMethod)
    cfg = config(FP8, non_routed_exl3={"bits": 5, "modules": ["o_proj"], "bf16_modules": ["gate"]})
    assert isinstance(_method(cfg, "model.layers.0.self_attn.o_proj"), EXL3LinearMethod)
    assert not isinstance(_method(cfg, "model.layers.0.mlp.gate"), FP8BlockLinearMethod)
    assert isinstance(_method(cfg, "model.layers.0.self_attn.qkv_proj"), FP8BlockLinearMethod)
    monkeypatch.setenv("SGLANG_EXL3_NON_ROUTED_FP8", "0")
    assert not isinstance(_method(cfg, "model.layers.0.self_attn.qkv_proj"), FP8BlockLinearMethod)


def test_routing_by_stored_tensors():
    def stored(module, *leaves):
        return {module: {"stored_tensors": {f"{module}.{leaf}": {"dtype": d} for leaf, d in leaves}}}

    pair = (("weight", "F8_E4M3"), ("weight_scale_inv", "F32"))
    ts = {**stored("model.language_model.layers.0.self_attn.o_proj", *pair),
          **stored("model.layers.0.mlp.gate_proj", *pair), **stored("model.layers.0.mlp.up_proj", *pair),
          **stored("model.layers.1.mlp.gate_proj", *pair), **stored("model.layers.1.mlp.up_proj", ("weight", "BF16")),
          **stored("model.layers.0.mlp.gate", ("weight", "BF16")),
          **stored("model.layers.0.odd", ("weight", "F8_E5M2"), ("weight_scale_inv", "F32")),
          **stored("model.layers.0.self_attn.q_proj", ("trellis", "I16"))}
    assert "model.layers.0.odd" not in fp8_block_modules(ts) and fp8_block_modules(None) == set()
    cfg = EXL3Config.from_config({"quant_method": "exl3", "bits": 3, "scope": "dense_and_moe", "tensor_storage": ts,
                                  "non_routed_quantization": FP8})
    for prefix in ("model.layers.0.self_attn.o_proj", "model.layers.0.mlp.gate_up_proj"):
        assert isinstance(_method(cfg, prefix), FP8BlockLinearMethod)
    for prefix in ("model.layers.1.mlp.gate_up_proj", "model.layers.0.mlp.gate", "model.layers.0.odd",
                   "model.layers.5.mlp.down_proj"):
        assert not isinstance(_method(cfg, prefix), FP8BlockLinearMethod)
    assert isinstance(_method(cfg, "model.layers.0.self_attn.q_proj"), EXL3LinearMethod)


@pytest.mark.parametrize("call", [
    ("exl3_fp8_quant_rows", P, 1 << 31, P, P, 1, 1, (1 << 30) + 16, None),
    ("exl3_fp8_quant_rows", P, 1 << 31, P, P, 1, 1, 0x7ffffff0, None),
    ("exl3_fp8_swiglu_quant", P, 1 << 32, 0.0, P, P, 1, 1, 0x7ffffff0, None),
    ("exl3_fp8_linear", P, 3, P, P, P, None, P, 1, (1 << 30) + 1, 16, 1, None, 0, None),
    ("exl3_fp8_linear", P, 3, P, P, P, None, P, 1, 1, 16, 0x7fffffff, None, 0, None),
    ("exl3_fp8_linear", P, 3, P, P, P, None, P, 1, 1, (1 << 22) + 16, 1, None, 0, None),
    ("exl3_fp8_linear", P, 3, P, P, P, None, P, 1, 1, 0x7ffffff0, 1, None, 0, None),
])
def test_abi_refuses_sizes_beyond_its_indexes(call):
    """Sizes at which a tile's indexes past the end would leave 32 bits."""
    L = _lib.lib()
    assert getattr(L, call[0])(*call[1:]) == _lib.EXL3_ERR_ARG
    assert b"above" in L.exl3_last_error() or b"too large" in L.exl3_last_error()


def test_swiglu_stride_counts_both_halves():
    """Twice the columns, also where that passes 31 bits."""
    L = _lib.lib()
    assert L.exl3_fp8_swiglu_quant(P, 1 << 30, 0.0, P, P, 1, 1, 1 << 30, None) == _lib.EXL3_ERR_ARG
    assert b"at least 2147483648" in L.exl3_last_error()
