"""8-bit base weights (``base_weights_fp8``, ``FusedLinear.quantize_fp8_``) and the 8-bit checkpoint store where the rest of the framework
meets them: merging, writing and loading checkpoints, configuration, moves between devices, adapters of several stacked projections, other
streams. Expected values come from the definitions in 64 bits."""
import pytest
import torch

from axolotl_b200.ops.fp8 import Fp8State

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, EPS32 = 2.0 ** -8, 2.0 ** -23


def _model(dev="cpu", layers=2, **kw):
    from axolotl_b200.models.config import preset
    from axolotl_b200.models.transformer import CausalLM

    cfg = preset("tiny-llama", num_hidden_layers=layers, vocab_size=512, **kw)
    return CausalLM(cfg, dtype=torch.bfloat16 if dev == "cuda" else torch.float32, device=dev).init_weights(0)


def _weight8(m):
    """The coded weight of a projection in 64 bits."""
    st = m.weight._axb_quant
    assert isinstance(st, Fp8State)
    N, K = m.weight.shape
    s = st.scale.cpu().double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return m.weight.data.view(torch.float8_e4m3fn).cpu().double() * s


# ------------------------------------------------------------------ checkpoints
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("quantize", ["fp8", "nf4"])
def test_merged_model_is_dense_everywhere(quantize, dev, tmp_path):
    """Adapters on some of the projections: merging expands the coded weights of the others too, and what is written reads back as the
    merged model. A coded weight is rounded to bf16 when it is expanded, and once more with the adapter's update in it."""
    from axolotl_b200.io.hf import load_pretrained, save_pretrained
    from axolotl_b200.models.lora import LoraSpec, inject_lora, merge_and_unload, quantize_base_fp8_, quantize_base_nf4_

    model = _model(dev)
    (quantize_base_fp8_ if quantize == "fp8" else quantize_base_nf4_)(model)
    torch.manual_seed(1)
    inject_lora(model, LoraSpec(r=8, lora_alpha=16, target_modules=["q_proj", "v_proj"]))
    want, delta = {}, {}
    for n, m in model.fused_linears():
        if not n.startswith("layers."):
            continue
        if m.lora_B is not None:
            with torch.no_grad():
                for _, B in m.peft_tensors().values():
                    B.normal_(0, 0.05)
            delta[n] = m.scaling * (m.lora_B.double() @ m.lora_A.double()).cpu().detach()
        want[n] = _weight8(m) if quantize == "fp8" else m._dense_weight().cpu().double()
    model.refresh_lora_shadows()
    assert 0 < len(delta) < len(want)
    merge_and_unload(model)
    save_pretrained(model, str(tmp_path / "m"))
    back = dict(load_pretrained(str(tmp_path / "m"), dtype=torch.float32, device="cpu").fused_linears())
    for n, m in model.fused_linears():
        if n not in want:
            continue
        assert m.weight.is_floating_point() and getattr(m.weight, "_axb_quant", None) is None, n
        assert torch.equal(m.weight.detach().float().cpu(), back[n].weight.detach()), n
        full = want[n] + delta.get(n, 0)
        tol = BF16 * (want[n].abs() + (full.abs() * (1 + BF16) if n in delta else 0)) + EPS32 * 16 * full.abs()
        assert ((m.weight.detach().cpu().double() - full).abs() <= tol).all(), n


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("preset_kw", [{}, dict(attention_bias=True)])
def test_written_weights_are_expanded(preset_kw, dev, tmp_path):
    """A model that is written while its projections are coded: every weight goes out as the values that the codes stand for."""
    from axolotl_b200.io.hf import hf_state_dict, load_pretrained, save_pretrained
    from axolotl_b200.models.lora import quantize_base_fp8_

    model = _model(dev, **preset_kw)
    quantize_base_fp8_(model)
    assert all(v.is_floating_point() for v in hf_state_dict(model).values())
    save_pretrained(model, str(tmp_path / "m"))
    back = dict(load_pretrained(str(tmp_path / "m"), dtype=torch.float32, device="cpu").fused_linears())
    for n, m in model.fused_linears():
        if n.startswith("layers."):
            w8 = _weight8(m)
            assert ((back[n].weight.detach().double() - w8).abs() <= (BF16 if dev == "cuda" else EPS32) * w8.abs()).all(), n


@pytest.mark.parametrize("quantize", ["fp8", "nf4"])
def test_loading_into_coded_weights_is_refused(quantize):
    """A checkpoint's values are no codes: a model takes them before it is coded, and the codes stay what they were."""
    from axolotl_b200.io.hf import hf_state_dict, load_state_into
    from axolotl_b200.models.lora import quantize_base_fp8_, quantize_base_nf4_

    model = _model()
    sd = {k: v.clone() for k, v in hf_state_dict(model).items()}
    load_state_into(model, sd.items())
    (quantize_base_fp8_ if quantize == "fp8" else quantize_base_nf4_)(model)
    before = {n: m.weight.data.clone() for n, m in model.fused_linears()}
    with pytest.raises(ValueError, match="codes"):
        load_state_into(model, sd.items())
    assert all(torch.equal(m.weight.data, before[n]) for n, m in model.fused_linears())
