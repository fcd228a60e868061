"""Which tensors of an artifact ``weight_dtype="int4"`` takes as they stand: those that the ``int4`` quantiser wrote, for the matrices that they are to be."""
import json

import pytest
import torch

from llmctl_b200.io.quantize import Int4GroupQuantizer


class Halved(Int4GroupQuantizer):
    """Writes bytes and scales of the same shapes under names of the same form, but the numbers are half as large."""
    name = "halved4"

    def dequantize(self, sd, dtype=torch.bfloat16):
        return {k: (v.float() * 0.5 if v.dim() == 2 and f"{k}.scale" in sd else v).to(v.dtype) for k, v in super().dequantize(sd, dtype).items()}


def _engine(artifact, **kw):
    from llmctl_b200.comms import mesh
    from llmctl_b200.serve.engine import InferenceEngine
    mesh.reset_state()
    torch.manual_seed(0)
    return InferenceEngine(artifact, device="cpu", kv_block_size=4, num_kv_blocks=64, max_batch_size=4, max_batch_tokens=512, **kw)


def _artifact(path, eng, quantiser):
    from safetensors.torch import save_file
    sd = quantiser.quantize({k: v.detach().clone() for k, v in eng.model.named_parameters()})
    (path / "model_config.json").write_text(json.dumps(eng.cfg.to_dict()))
    (path / "export.json").write_text(json.dumps({"quantization": quantiser.name}))
    save_file({k: v.contiguous() for k, v in sd.items()}, str(path / "model.safetensors"))
    return sd


@pytest.fixture
def _registered():
    from llmctl_b200.plugins.registry import get_registry
    get_registry().register("quantizers", "halved4", Halved, overwrite=True)
    yield
    get_registry()._items["quantizers"].pop("halved4")


def test_codes_of_another_scheme_are_not_taken_for_its_own(tmp_path, _registered):
    plain = _engine("gpt-tiny")
    _artifact(tmp_path, plain, Halved())
    loaded, held = _engine(str(tmp_path)), _engine(str(tmp_path), weight_dtype="int4")
    x = torch.tensor([[5, 6, 7, 200, 9]])
    with torch.no_grad():
        want, got = loaded.model(x), held.model(x)
    assert (got - want).norm() / want.norm() < 0.2 < (plain.model(x) - want).norm() / want.norm()


def test_codes_that_do_not_fit_are_not_taken():
    from llmctl_b200.models.int4 import Int4Linear, hold_in_int4
    sd = Int4GroupQuantizer().quantize({k: v.detach().clone() for k, v in _engine("gpt-tiny").model.named_parameters()})
    name = next(k for k in sd if k.endswith("qkv.weight"))
    for bad in ({name: sd[name][:-4], name + ".scale": sd[name + ".scale"][:-4]}, {name: sd[name], name + ".scale": sd[name + ".scale"].float()},
                {name: torch.cat([sd[name], sd[name]], 1), name + ".scale": sd[name + ".scale"]}, {name: sd[name]}):
        model = _engine("gpt-tiny").model
        assert hold_in_int4(model, {k: v for k, v in {**sd, **bad}.items() if len(bad) == 2 or k != name + ".scale"}) > 0
        layer = model.get_submodule(name.rpartition(".")[0])
        assert isinstance(layer, Int4Linear) and torch.equal(layer.weight, sd[name]) and torch.equal(layer.scale, sd[name + ".scale"])


@pytest.mark.parametrize("quantised", [True, False])
def test_an_artifact_is_read_once(tmp_path, monkeypatch, quantised):
    import safetensors.torch
    eng = _engine("gpt-tiny")
    if quantised:
        _artifact(tmp_path, eng, Int4GroupQuantizer())
    else:
        (tmp_path / "model_config.json").write_text(json.dumps(eng.cfg.to_dict()))
        safetensors.torch.save_file({k: v.detach().clone() for k, v in eng.model.named_parameters()}, str(tmp_path / "model.safetensors"))
    reads, read = [], safetensors.torch.load_file
    monkeypatch.setattr(safetensors.torch, "load_file", lambda *a, **k: (reads.append(a[0]), read(*a, **k))[1])
    held = _engine(str(tmp_path), weight_dtype="int4")
    assert len(reads) == 1
    assert held.generate([[5, 6, 7]], max_tokens=4, temperature=0.0) == _engine("gpt-tiny", weight_dtype="int4").generate([[5, 6, 7]], max_tokens=4, temperature=0.0)


def test_a_projection_gives_its_weights_back_as_it_is_replaced(monkeypatch):
    """While a model is rounded, never more than one of its wide matrices stands beside those that are still to come."""
    import weakref
    from llmctl_b200.models import int4
    model, seen, alive = _engine("gpt-tiny").model, [], []
    quantise = int4.Int4GroupQuantizer.quantize

    def watched(self, sd):
        alive.append(sum(r() is not None for r in seen))
        seen.extend(weakref.ref(model.get_submodule(k.removesuffix(".weight"))) for k in sd)
        return quantise(self, sd)

    monkeypatch.setattr(int4.Int4GroupQuantizer, "quantize", watched)
    replaced = int4.hold_in_int4(model)
    assert len(seen) == replaced > 4 and max(alive) <= 1
