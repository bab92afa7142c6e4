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


# ------------------------------------------------------------------ the checkpoint store on several streams
def _values(x):
    from axolotl_b200.ops.fp8 import dequantize_fp8_rows, quantize_fp8_rows

    return dequantize_fp8_rows(*quantize_fp8_rows(x)) if x.dtype == torch.bfloat16 else x.clone()


@pytest.mark.gpu
@pytest.mark.parametrize("coded", [True, False])
@pytest.mark.parametrize("producer,consumer", [("default", "side"), ("side", "default"), ("side", "other")])
def test_store_waits_for_the_stream_that_wrote(producer, consumer, coded):
    """Only the producing stream is behind: some 25 ms of sleep lie before the tensor and its codes are written, none before they are taken
    back. The memory that the codes come to lie in holds other bytes before."""
    from axolotl_b200.train.activation_memory import make_store

    streams = {"default": torch.cuda.default_stream(), "side": torch.cuda.Stream(), "other": torch.cuda.Stream()}
    src, dst = streams[producer], streams[consumer]
    g = torch.Generator().manual_seed(1)
    x = torch.randn(512, 1024, generator=g).bfloat16().cuda()
    x = x if coded else x.double()
    want, store = _values(x), make_store("fp8", x.device)
    with torch.cuda.stream(src):
        late = torch.full_like(x, 3.0)
        scrap = [torch.full((n,), 0x38, dtype=torch.uint8, device="cuda") for n in (512 * 1024 + 8 * 512 * 4, 512 * 1024 * 8)]
    torch.cuda.synchronize()
    del scrap
    with torch.cuda.stream(src):
        torch.cuda._sleep(50_000_000)
        late.copy_(x)
        h = store.put(late)
    with torch.cuda.stream(dst):
        got = store.get(h).clone()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("coded", [True, False])
@pytest.mark.parametrize("producer", ["default", "side"])
def test_store_keeps_its_memory_while_another_stream_reads(producer, coded):
    """The producer has ended, the consumer is behind: the codes' memory is not given out again before the consumer has read it."""
    from axolotl_b200.train.activation_memory import make_store

    src, dst = torch.cuda.default_stream() if producer == "default" else torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.randn(512, 1024, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    x = x if coded else x.double()
    want, store = _values(x), make_store("fp8", x.device)
    torch.cuda.synchronize()
    with torch.cuda.stream(src):
        late = x.clone()
        h = store.put(late)
        size = h.gpu.numel() * h.gpu.element_size()
        del late
    src.synchronize()
    with torch.cuda.stream(dst):
        torch.cuda._sleep(50_000_000)
        got = store.get(h).clone()
    with torch.cuda.stream(src):
        fresh = [torch.full((size,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and fresh


@pytest.mark.gpu
def test_store_on_two_streams_of_one_captured_graph():
    """Put on the capturing stream and taken back on one that it forks, every replay with new values."""
    from axolotl_b200.train.activation_memory import make_store

    x = torch.zeros(300, 520, dtype=torch.bfloat16, device="cuda")
    store, side = make_store("fp8", x.device), torch.cuda.Stream()
    _values(x)
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        h = store.put(x)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out.copy_(store.get(h))
        torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        assert torch.equal(out, _values(x))


# ------------------------------------------------------------------ dependent launches
@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N", [(40, 8192, 512), (300, 2048, 1024), (2100, 1024, 2600)])
def test_products_see_the_rows_of_the_launch_before_them(T, K, N):
    """Codes and scales of one call lie where those of the call before lay, and their scales are far apart: a product, which starts while its
    rows are still being quantised, gives for each what it gives alone."""
    from axolotl_b200.ops import fp8

    g = torch.Generator().manual_seed(T)
    w, ws = fp8.quantize_fp8_weight(torch.randn(N, K, generator=g).cuda())
    rows = [(torch.randn(T, K, generator=g) * 2.0 ** e).bfloat16().cuda() for e in (0, -20, 20, 7)]
    alone = []
    for x in rows:
        alone.append(fp8._product(x, w, ws, keep=True)[0])
        torch.cuda.synchronize()
    torch.cuda.empty_cache()
    together = [fp8._product(rows[i % 4], w, ws, keep=True)[0] for i in range(32)]
    torch.cuda.synchronize()
    for i, y in enumerate(together):
        assert torch.equal(y, alone[i % 4]), i


# ------------------------------------------------------------------ rows of whole 16 bytes
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("K", [2008, 200, 256])
def test_codes_keep_their_row_layout_when_they_move(K, dev):
    """Rows of codes start on 16 bytes as they were laid out when the weight was quantised, wherever the module goes: no product lays the
    weight out again."""
    from axolotl_b200.models.layers import FusedLinear
    from axolotl_b200.ops import fp8

    m = FusedLinear(K, [40], ["a"], dtype=torch.float32, device="cpu")
    with torch.no_grad():
        m.weight.copy_(torch.randn(40, K, generator=torch.Generator().manual_seed(1)))
    m.quantize_fp8_()
    codes, scale = m.weight.data.clone(), m.weight._axb_quant.scale.clone()
    moves = [lambda: m._apply(lambda t: t.clone(memory_format=torch.contiguous_format)), lambda: m.to(dev), lambda: m.to(torch.bfloat16),
             lambda: m.cpu(), lambda: m.to(dev)]
    for move in moves:
        move()
        w = m.weight
        assert w.stride(1) == 1 and w.stride(0) % 16 == 0 and w.data_ptr() % 16 == 0 and not w.requires_grad
        assert torch.equal(w.data.cpu(), codes) and torch.equal(w._axb_quant.scale.cpu(), scale) and w._axb_quant.scale.device == w.device
        assert fp8._rows16(w.data.view(torch.float8_e4m3fn)).data_ptr() == w.data_ptr()


@pytest.mark.parametrize("dev", DEVICES)
def test_codes_keep_their_row_layout_under_layer_offloading(dev):
    """The host copy has the rows' padding, and so has what comes back."""
    from axolotl_b200.models.lora import LoraSpec, inject_lora, quantize_base_fp8_
    from axolotl_b200.train.activation_memory import LayerOffloader

    m = _model(dev, layers=3, intermediate_size=200)          # down: rows of 200 codes
    quantize_base_fp8_(m)
    inject_lora(m, LoraSpec(r=8, lora_alpha=16, target_modules=["q_proj"]))
    ids = torch.randint(0, 512, (1, 32), generator=torch.Generator().manual_seed(2)).to(dev)
    want = m(ids, labels=ids).loss.item()
    seen = []
    off = LayerOffloader(m, dev)
    for layer in m.layers:
        w = layer.mlp.down_proj.weight
        assert w.numel() == 0
        layer.mlp.down_proj.register_forward_pre_hook(lambda mod, a: seen.append((tuple(mod.weight.shape), mod.weight.stride())))
    loss = m(ids, labels=ids).loss
    loss.backward()
    assert loss.item() == want and seen and all(shape[1] == 200 and stride == (208, 1) for shape, stride in seen)
    assert off.bytes_per_layer


# ------------------------------------------------------------------ configuration
BASE = {"model_preset": "tiny-llama", "adapter": "lora", "lora_r": 8, "lora_alpha": 16, "lora_target_linear": True, "sequence_len": 64,
        "micro_batch_size": 1, "gradient_accumulation_steps": 1, "max_steps": 1, "learning_rate": 1e-3, "output_dir": "unused",
        "device": "cpu", "datasets": [{"path": "synthetic", "type": "_synthetic"}], "base_weights_fp8": True}


def test_restarts_that_fold_into_codes_are_refused():
    from axolotl_b200.config.load import load_cfg

    relora = {"relora": True, "jagged_restart_steps": 100}
    with pytest.raises(ValueError, match="base_weights_fp8"):
        load_cfg({**BASE, **relora})
    assert load_cfg({**BASE, **relora, "base_weights_fp8": False})["relora"]


@pytest.mark.parametrize("key,bad,good", [
    ("unfrozen_parameters", [r"layers\.1\.mlp\.down_proj"], [r"layers\.\d+\.input_layernorm", "embed_tokens"]),
    ("unfrozen_parameters", ["embed_tokens", r"^layers\.0\."], ["^norm"]),
    ("unfrozen_parameters", [r"qkv_proj\.weight$"], [r"qkv_proj\.bias$"]),
    ("unfrozen_parameters", [r"layers\.37\.self_attn\.kv_b_proj"], ["lm_head"]),
    ("lora_modules_to_save", ["down_proj"], ["embed_tokens", "lm_head"]),
    ("lora_modules_to_save", ["mlp"], ["layernorm"])])
def test_training_a_coded_projection_is_refused(key, bad, good):
    """Codes take no gradient: what would train them is refused with the configuration, before a model is loaded."""
    from axolotl_b200.config.load import load_cfg

    with pytest.raises(ValueError, match="base_weights_fp8"):
        load_cfg({**BASE, key: bad})
    assert list(load_cfg({**BASE, key: good})[key]) == good
    assert list(load_cfg({**BASE, "base_weights_fp8": False, key: bad})[key]) == bad


def test_training_a_coded_projection_is_refused_by_its_own_name():
    """A plugin may name parameters after the configuration was checked, and a family may have projections of other names: the model's own
    names are checked before a weight is coded."""
    from axolotl_b200.config.load import load_cfg
    from axolotl_b200.train.run import setup_adapter

    model = _model()
    model.layers[1].other_proj, model.layers[1].mlp.down_proj = model.layers[1].mlp.down_proj, None
    cfg = load_cfg(dict(BASE))
    cfg["unfrozen_parameters"] = ["other_proj"]
    with pytest.raises(ValueError, match="layers.1.other_proj.weight"):
        setup_adapter(cfg, model)
    assert all(m.weight.is_floating_point() for _, m in model.fused_linears())


# ------------------------------------------------------------------ rows in fp16
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("K", [264, 131])
def test_finite_values_of_fp16_stay_finite(K, dev):
    """From 248 * 2^8 on the nearest code stands for 2^16, which fp16 does not have: its largest number comes back, half a step of E4M3 off
    at most. What is further beyond overflows as in any conversion."""
    from axolotl_b200.ops.fp8 import dequantize_fp8_rows, quantize_fp8_rows
    from axolotl_b200.train.activation_memory import make_store

    x = torch.zeros(3, K, dtype=torch.float16)
    x[0, :6] = torch.tensor([65504.0, -65504.0, 63488.0, 63456.0, -61440.0, 3.0])
    x[1, 128:131] = torch.tensor([-65504.0, 1.0, 65472.0])
    x[2, 0] = float("inf")
    want = x.clone()
    want[0, :6] = torch.tensor([65504.0, -65504.0, 65504.0, 61440.0, -61440.0, 3.0])     # 248 lies in the middle: to even, 256; scale 2^8
    want[1, 128:131] = torch.tensor([-65504.0, 1.0, 65504.0])
    codes, scale = quantize_fp8_rows(x.to(dev))
    back = dequantize_fp8_rows(codes, scale, torch.float16).cpu()
    assert torch.isnan(back[2, 0]) and back[2, 1:].abs().sum() == 0 and torch.equal(back[:2], want[:2])
    assert dequantize_fp8_rows(codes, scale, torch.float32)[0, 0].item() == 65536.0       # what the code stands for
    store = make_store("fp8", dev)
    assert torch.equal(store.get(store.put(x.to(dev)))[:2].cpu(), want[:2])
    big = torch.full((1, K), 1e5, dtype=torch.float32, device=dev)
    assert torch.isinf(dequantize_fp8_rows(*quantize_fp8_rows(big), dtype=torch.float16)).all()


# ------------------------------------------------------------------ arguments
@pytest.mark.parametrize("dev", DEVICES)
def test_half_an_extension_is_refused(dev):
    from axolotl_b200.ops.fp8 import fp8_gemm, quantize_fp8_rows, quantize_fp8_weight

    codes, scale = quantize_fp8_rows(torch.ones(4, 128, device=dev).bfloat16())
    w, ws = quantize_fp8_weight(torch.ones(64, 128, device=dev))
    for kw in (dict(b2=torch.zeros(64, 8, device=dev).bfloat16()), dict(a2=torch.zeros(4, 8, device=dev).bfloat16())):
        with pytest.raises(ValueError, match="extension"):
            fp8_gemm(codes, scale, w, ws, **kw)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [1, 70, 200])
def test_adapter_gradient_of_rows_in_any_layout(T, dev):
    """t as one row for all tokens, as overlapping rows, as columns of a wider matrix and transposed: what it gives laid out plainly. The
    factors are small integers and the rows their own codes, so that every sum is exact."""
    from axolotl_b200.ops.fp8 import fp8_adapter_grad, quantize_fp8_rows

    g = torch.Generator().manual_seed(T)
    x = torch.randint(-2, 3, (T, 264), generator=g).bfloat16().to(dev)
    codes, scale = quantize_fp8_rows(x)
    flat = torch.randint(-2, 3, (T * 40 + 64,), generator=g).bfloat16().to(dev)
    for t in (flat[:16].expand(T, 16), flat.as_strided((T, 16), (8, 1)), flat[:T * 40].view(T, 40)[:, 3:19],
              flat[:T * 16].view(16, T).t(), flat[:1].expand(T, 1), flat[:T * 9].view(T, 9)):
        want = t.cpu().double().t() @ x.cpu().double()
        assert torch.equal(fp8_adapter_grad(t, codes, scale).cpu().double(), want), t.stride()
        out = torch.ones(want.shape, device=dev)
        assert torch.equal(fp8_adapter_grad(t, codes, scale, out=out).cpu().double(), want + 1)


# ------------------------------------------------------------------ adapters
def _rows8(x):
    from axolotl_b200.ops.fp8 import dequantize_fp8_rows, quantize_fp8_rows

    return dequantize_fp8_rows(*quantize_fp8_rows(x.cpu()), dtype=torch.float32).double()


def _adapter(N, K, blocks, seed=1):
    """(A, B) in fp32 with bf16 values, B block diagonal."""
    g = torch.Generator().manual_seed(seed)
    R = sum(b[3] for b in blocks)
    A, B = (torch.randn(R, K, generator=g) * K ** -0.5).bfloat16().float(), torch.zeros(N, R)
    for r0, rows, c0, r in blocks:
        B[r0:r0 + rows, c0:c0 + r] = (torch.randn(rows, r, generator=g) * 0.1).bfloat16().float()
    return A, B


QKV = ((0, 256, 0, 16), (256, 64, 16, 16), (320, 64, 32, 16))                    # q | k | v, rank 16 each
ADAPTERS = [(1, 264, 384, QKV), (513, 264, 384, QKV), (960, 520, 640, ((0, 640, 0, 16),)), (700, 136, 264, ((0, 100, 0, 3), (100, 150, 3, 5))),
            (130, 264, 520, ((0, 264, 0, 32), (264, 256, 32, 32))), (8192, 136, 128, ((0, 128, 0, 8),)), (8200, 136, 264, ((8, 200, 0, 8),)),
            (17000, 136, 384, QKV)]


@pytest.mark.gpu
@pytest.mark.parametrize("masters", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,N,blocks", ADAPTERS)
def test_adapter_gradients_repeat_and_are_what_they_are(T, K, N, blocks, masters):
    """The sums over column ranges and row chunks are joined in one order: the same bits every time. Against 64 bits: s x A^T and s dy B are
    held in bf16 (2^-8 of themselves and their sums in fp32), each sum of n products is off by n 2^-23 of the sum of magnitudes."""
    from axolotl_b200.ops.fp8 import fp8_lora_linear, quantize_fp8_weight

    g = torch.Generator().manual_seed(T)
    x, dy = torch.randn(T, K, generator=g).bfloat16(), (torch.randn(T, N, generator=g) * 1e-2).bfloat16()
    w, ws = quantize_fp8_weight(torch.randn(N, K, generator=g).cuda())
    A, B = _adapter(N, K, blocks)
    leaves = [x.cuda().requires_grad_(True)] + [t.to(masters).cuda().requires_grad_(True) for t in (A, B)]
    A16, B16 = A.bfloat16().cuda(), B.bfloat16().cuda()
    runs = []
    for _ in range(4):
        y = fp8_lora_linear(leaves[0], w, ws, leaves[1], leaves[2], A16, B16, 2.0, blocks)
        runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy.cuda())])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))
    y, dx, dA, dB = (t.cpu().double() for t in runs[0])
    a, b, x64, d64, x8 = A.double(), B.double(), x.double(), dy.double(), _rows8(x)
    low, tall = 2 * x64 @ a.t(), 2 * d64 @ b
    low_e = BF16 * low.abs() + (K + 2) * EPS32 * 2 * x64.abs() @ a.abs().t()
    tall_e = BF16 * tall.abs() + (N + 2) * EPS32 * 2 * d64.abs() @ b.abs()
    half = BF16 if masters == torch.bfloat16 else 0.0
    for got, want, off, size in ((dA, tall.t() @ x8, tall_e.t() @ x8.abs(), tall.abs().t() @ x8.abs()),
                                 (dB, d64.t() @ low, d64.abs().t() @ low_e, d64.abs().t() @ low.abs())):
        tol = half * (1 + BF16) * want.abs() + (1 + half) * off + (T + 32) * EPS32 * size
        if got is dB:
            inside = torch.zeros(N, B.shape[1], dtype=torch.bool)
            for r0, rows, c0, r in blocks:
                inside[r0:r0 + rows, c0:c0 + r] = True
            assert (got[~inside] == 0).all()
            want, tol = want * inside, tol * inside
        assert ((got - want).abs() <= tol + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [300, 8200])
@pytest.mark.parametrize("shift", [0, 1])
def test_adapter_gradients_add_to_flat_buffers_in_order(T, shift):
    """Gradients that are added where the optimizer keeps them, at any address: twice the same pass is one pass and its own sum, and what
    lies beside the buffer and outside the blocks stays."""
    from axolotl_b200.ops.fp8 import fp8_lora_linear, quantize_fp8_weight

    K, N, R = 264, 384, 48
    g = torch.Generator().manual_seed(T)
    x, dy = torch.randn(T, K, generator=g).bfloat16().cuda(), (torch.randn(T, N, generator=g) * 1e-2).bfloat16().cuda()
    w, ws = quantize_fp8_weight(torch.randn(N, K, generator=g).cuda())
    A, B = (t.cuda().requires_grad_(True) for t in _adapter(N, K, QKV))
    A16, B16 = A.detach().bfloat16(), B.detach().bfloat16()
    fresh = torch.autograd.grad(fp8_lora_linear(x, w, ws, A, B, A16, B16, 2.0, QKV), [A, B], dy)
    for start in (0.0, 3.0):
        flat = [torch.full((t.numel() + 2,), start, device="cuda") for t in (A, B)]
        A._axb_grad, B._axb_grad = (f[shift:shift + t.numel()].view(t.shape) for f, t in zip(flat, (A, B)))
        torch.autograd.backward(fp8_lora_linear(x, w, ws, A, B, A16, B16, 2.0, QKV), dy)
        for f, got, t in zip(flat, (A._axb_grad, B._axb_grad), fresh):
            # the sum is added at once, or (more than 8192 rows of dB) in two parts: one rounding each
            tol = EPS32 * 2 * (t.abs() + start) if start or T > 8192 else torch.zeros_like(t)
            assert ((got - t - start).abs() <= tol).all()
            assert (f[:shift] == start).all() and (f[shift + t.numel():] == start).all()
        outside = torch.ones(N, R, dtype=torch.bool, device="cuda")
        for r0, rows, c0, r in QKV:
            outside[r0:r0 + rows, c0:c0 + r] = False
        assert (B._axb_grad[outside] == start).all()
    del A._axb_grad, B._axb_grad


@pytest.mark.gpu
def test_adapter_layer_on_a_second_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    from axolotl_b200.ops.fp8 import fp8_lora_linear, quantize_fp8_weight

    got = []
    for dev in ("cuda:0", "cuda:1"):
        g = torch.Generator().manual_seed(1)
        x, dy = torch.randn(70, 264, generator=g).bfloat16().to(dev).requires_grad_(True), torch.randn(70, 384, generator=g).bfloat16().to(dev)
        w, ws = quantize_fp8_weight(torch.randn(384, 264, generator=g).to(dev))
        A, B = (t.to(dev).requires_grad_(True) for t in _adapter(384, 264, QKV))
        y = fp8_lora_linear(x, w, ws, A, B, A.detach().bfloat16(), B.detach().bfloat16(), 2.0, QKV)
        got.append([t.cpu() for t in (y, *torch.autograd.grad(y, [x, A, B], dy))])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,blocks", [(1, 136, 384, QKV), (40, 4096, 256, ((0, 256, 0, 64),)), (520, 264, 640, ((0, 640, 0, 16),)),
                                          (700, 2056, 384, QKV), (1000, 14336, 256, ((0, 256, 0, 32),)), (8300, 136, 264, ((0, 264, 0, 8),))])
def test_adapter_gradients_see_the_sums_in_sixteen_bits(T, K, N, blocks):
    """dA and dB of fp32 masters: s dy B and s x A^T enter as two bf16 numbers, which are off by 2^-16 of the value together, so that what is
    left is the sums' own error in fp32."""
    from axolotl_b200.ops.fp8 import fp8_lora_linear, quantize_fp8_weight

    g = torch.Generator().manual_seed(T)
    x, dy = torch.randn(T, K, generator=g).bfloat16(), (torch.randn(T, N, generator=g) * 1e-2).bfloat16()
    w, ws = quantize_fp8_weight(torch.randn(N, K, generator=g).cuda())
    A, B = _adapter(N, K, blocks)
    Al, Bl = A.cuda().requires_grad_(True), B.cuda().requires_grad_(True)
    y = fp8_lora_linear(x.cuda(), w, ws, Al, Bl, A.bfloat16().cuda(), B.bfloat16().cuda(), 2.0, blocks)
    dA, dB = (t.cpu().double() for t in torch.autograd.grad(y, [Al, Bl], dy.cuda()))
    a, b, x64, d64, x8 = A.double(), B.double(), x.double(), dy.double(), _rows8(x)
    low, tall = 2 * x64 @ a.t(), 2 * d64 @ b
    low_e = 2.0 ** -16 * low.abs() + (K + 16) * EPS32 * 2 * x64.abs() @ a.abs().t()
    tall_e = 2.0 ** -16 * tall.abs() + (N + 160) * EPS32 * 2 * d64.abs() @ b.abs()          # parts of up to 148 column ranges
    assert ((dA - tall.t() @ x8).abs() <= tall_e.t() @ x8.abs() + (2 * T + 32) * EPS32 * tall.abs().t() @ x8.abs() + 1e-30).all()
    for r0, rows, c0, r in blocks:
        d, l, e = d64[:, r0:r0 + rows], low[:, c0:c0 + r], low_e[:, c0:c0 + r]
        assert ((dB[r0:r0 + rows, c0:c0 + r] - d.t() @ l).abs() <= d.abs().t() @ e + (2 * T + 64) * EPS32 * d.abs().t() @ l.abs() + 1e-30).all()


# ------------------------------------------------------------------ profiles
def test_every_kernel_of_the_8_bit_blocks_has_a_category():
    import pathlib
    import re

    import axolotl_b200
    from axolotl_b200.utils.analyze_profile import categorize

    names = set()
    for f in sorted((pathlib.Path(axolotl_b200.__file__).parent / "csrc").glob("fp8_*.cu")):
        names |= set(re.findall(r"\b(fp8_\w+_kernel)\s*\(", f.read_text()))
    assert len(names) >= 6
    for n in names:
        where = [c for c, (count, _) in categorize([(f"void (anonymous namespace)::{n}<16, true>(...)", 1.0)]).items() if count]
        assert where in (["8-bit products"], ["8-bit rows"]), n


@pytest.mark.gpu
@pytest.mark.parametrize("K", [264, 14336])
def test_infinities_stay_infinities_in_the_gradient_of_b(K):
    """An infinite x A^T has nothing that bf16 leaves of it: dB is infinite where the formula says so, and no NaN."""
    from axolotl_b200.ops.fp8 import fp8_lora_linear, quantize_fp8_weight

    T, N, R = 200, 128, 16
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(T, K, generator=g).bfloat16(), torch.randn(T, N, generator=g).bfloat16()
    dy[dy == 0] = 1
    x[77, 5] = float("inf")
    w, ws = quantize_fp8_weight(torch.randn(N, K, generator=g).cuda())
    A, B = _adapter(N, K, ((0, N, 0, R),))
    A[:, 5] = torch.where(A[:, 5] == 0, 1.0, A[:, 5])
    B0 = B.cuda().requires_grad_(True)
    y = fp8_lora_linear(x.cuda(), w, ws, A.cuda(), B0, A.bfloat16().cuda(), B.bfloat16().cuda(), 2.0, ((0, N, 0, R),))
    (dB,) = torch.autograd.grad(y, [B0], dy.cuda())
    want = dy[77].double()[:, None].sign() * A.double()[:, 5].sign()[None] * float("inf")
    assert torch.equal(dB.cpu().double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,R", [(64, 14336, 16), (64, 2048, 48), (700, 8192, 48), (700, 8192, 8), (2000, 4096, 64), (2000, 4096, 8)])
def test_one_pass_and_two_keep_the_same(T, K, R):
    """On both sides of the rule that picks one pass over x or two: the codes are the quantiser's, s x A^T is its sum to 2^-16 of itself."""
    from axolotl_b200.ops.fp8 import _unpacked, fp8_lora_linear, quantize_fp8_rows, quantize_fp8_weight

    g = torch.Generator().manual_seed(T + R)
    x = torch.randn(T, K, generator=g).bfloat16().cuda()
    A, B = _adapter(64, K, ((0, 64, 0, R),))
    w, ws = quantize_fp8_weight(torch.randn(64, K, generator=g).cuda())
    A, B = A.cuda().requires_grad_(True), B.cuda().requires_grad_(True)
    y = fp8_lora_linear(x, w, ws, A, B, A.detach().bfloat16(), B.detach().bfloat16(), 0.5, ((0, 64, 0, R),))
    q, xa = y.grad_fn.saved_tensors[0], y.grad_fn.saved_tensors[7]
    (c, s), (codes, scale) = _unpacked(q, T, K), quantize_fp8_rows(x)
    assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s, scale) and xa.shape == (2, T, R)
    want, size = 0.5 * x.double() @ A.double().t(), 0.5 * x.double().abs() @ A.double().abs().t()
    assert ((xa.double().sum(0) - want).abs() <= 2.0 ** -16 * want.abs() + (K + 16) * EPS32 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 50, 960])
@pytest.mark.parametrize("names,outs,r", [(["q_proj", "k_proj", "v_proj"], [512, 128, 128], 16), (["gate_proj", "up_proj"], [704, 704], 16),
                                          (["q_proj", "k_proj", "v_proj"], [264, 72, 72], 8), (["o_proj"], [520], 64)])
def test_stacked_adapters_of_a_coded_projection(T, names, outs, r):
    """A fused projection as a model has it: the adapters of q | k | v (rank 48 for 16 each) or gate | up stacked, B block diagonal, fp32
    masters with bf16 copies, gradients into the masters or into flat buffers. Against the definition in 64 bits."""
    from axolotl_b200.models.layers import FusedLinear

    K, N = 520, sum(outs)
    g = torch.Generator().manual_seed(T)
    m = FusedLinear(K, outs, names, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        m.weight.copy_(torch.randn(N, K, generator=g))
    m.quantize_fp8_()
    m.add_lora(r, 2 * r, targets=names)
    with torch.no_grad():
        for A, B in m.peft_tensors().values():
            B.copy_(torch.randn(B.shape, generator=g) * 0.1)
    m.refresh_shadows()
    m.train()
    assert m.lora_A.dtype == torch.float32 and m.lora_A.shape == (r * len(names), K) and len(m.lora_blocks) == len(names)
    x, dy = torch.randn(T, K, generator=g).bfloat16(), (torch.randn(T, N, generator=g) * 1e-2).bfloat16()
    xl = x.cuda().requires_grad_(True)
    y = m(xl)
    dx, dA, dB = torch.autograd.grad(y, [xl, m.lora_A, m.lora_B], dy.cuda())
    a, b = m.lora_A16.cpu().double(), m.lora_B16.cpu().double()
    w8, x64, d64, x8, d8, R = _weight8(m), x.double(), dy.double(), _rows8(x), _rows8(dy), a.shape[0]
    low, tall = m.scaling * x64 @ a.t(), m.scaling * d64 @ b
    low_s, tall_s = (K + 16) * EPS32 * m.scaling * x64.abs() @ a.abs().t(), (N + 160) * EPS32 * m.scaling * d64.abs() @ b.abs()
    for got, want, off, size, n in (
            (y, x8 @ w8.t() + low @ b.t(), (BF16 * low.abs() + low_s) @ b.abs().t(), x8.abs() @ w8.abs().t() + low.abs() @ b.abs().t(), K),
            (dx, d8 @ w8 + tall @ a, (BF16 * tall.abs() + tall_s) @ a.abs(), d8.abs() @ w8.abs() + tall.abs() @ a.abs(), N)):
        tol = BF16 * want.abs() + (1 + BF16) * (off + (n + R + 64) * EPS32 * size)
        assert ((got.detach().cpu().double() - want).abs() <= tol + 1e-30).all()
    assert ((dA.cpu().double() - tall.t() @ x8).abs() <= (2.0 ** -16 * tall.abs() + tall_s).t() @ x8.abs()
            + (2 * T + 32) * EPS32 * tall.abs().t() @ x8.abs() + 1e-30).all()
    inside = torch.zeros(N, R, dtype=torch.bool)
    for r0, rows, c0, k in m.lora_blocks:
        inside[r0:r0 + rows, c0:c0 + k] = True
    offB = d64.abs().t() @ (2.0 ** -16 * low.abs() + low_s) + (2 * T + 64) * EPS32 * d64.abs().t() @ low.abs() + 1e-30
    assert ((dB.cpu().double() - d64.t() @ low).abs() <= offB)[inside].all() and not dB.cpu()[~inside].any()
    m.lora_A._axb_grad, m.lora_B._axb_grad = torch.zeros_like(m.lora_A), torch.zeros_like(m.lora_B)
    xl.grad = None
    m(xl).backward(dy.cuda())
    assert m.lora_A.grad is None and torch.equal(m.lora_A._axb_grad, dA) and torch.equal(m.lora_B._axb_grad, dB) and torch.equal(xl.grad, dx)


def test_few_tokens_take_the_form_that_measured_best():
    """Forms that were timed side by side among other calls (tokens, rows of codes, columns): inside the product up to 12 blocks a CTA and pass,
    before it from 14 on, by tiles where more than 32 tokens meet enough of them."""
    from axolotl_b200.ops.fp8 import _few

    for form, shapes in ((2, [(1, 4096, 4096), (1, 2048, 8192), (24, 11264, 2048), (24, 4096, 4096), (48, 2048, 2048), (64, 2048, 2048)]),
                         (1, [(1, 4096, 14336), (16, 4096, 14336), (24, 6144, 4096), (24, 2048, 8192), (48, 4096, 4096), (64, 4096, 4096),
                              (1, 28672, 4096), (64, 4096, 14336), (64, 6144, 4096)]),
                         (0, [(48, 11264, 2048), (64, 28672, 4096), (65, 4096, 4096)])):
        for shape in shapes:
            assert _few(*shape) == form, shape


# ------------------------------------------------------------------ copies of modules
def _coded_linear(dev, K=200, quantize="fp8", seed=1):
    from axolotl_b200.models.layers import FusedLinear

    m = FusedLinear(K, [64, 24], ["a", "b"], bias=True, dtype=torch.bfloat16 if dev == "cuda" else torch.float32, device=dev)
    with torch.no_grad():
        m.weight.copy_(torch.randn(88, K, generator=torch.Generator().manual_seed(seed)))
    m.quantize_fp8_() if quantize == "fp8" else m.quantize_nf4_()
    return m


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("quantize,K", [("fp8", 200), ("fp8", 256), ("nf4", 256)])
def test_a_copied_module_keeps_what_its_codes_stand_for(quantize, K, dev):
    import copy
    import io

    m = _coded_linear(dev, K, quantize)
    m.add_lora(8, 16, targets=["b"])
    m.refresh_shadows()
    x = torch.randn(5, K, generator=torch.Generator().manual_seed(2)).to(dev, m.bias.dtype)
    want, buf = m(x), io.BytesIO()
    torch.save(m, buf)
    buf.seek(0)
    box = torch.nn.Module()
    box.a = box.b = m
    twice = copy.deepcopy(box)
    assert twice.a is twice.b
    for c in (copy.deepcopy(m), twice.a, torch.load(buf, weights_only=False)):
        assert torch.equal(c(x), want) and not c.weight.requires_grad and c.weight.data_ptr() != m.weight.data_ptr()
        assert c.weight._axb_quant is not m.weight._axb_quant
        if quantize == "fp8":
            assert c.weight.stride(0) % 16 == 0 and c.weight._axb_quant.scale.data_ptr() != m.weight._axb_quant.scale.data_ptr()


@pytest.mark.parametrize("dev", DEVICES)
def test_state_dicts_hold_the_scales_of_the_codes(dev):
    """Codes go from a coded module to a coded one with their scales; values and codes are not copied over one another."""
    a, b = _coded_linear(dev, seed=1), _coded_linear(dev, seed=2)
    x = torch.randn(5, 200, generator=torch.Generator().manual_seed(2)).to(dev, a.bias.dtype)
    assert not torch.equal(a(x), b(x))
    sd = a.state_dict()
    assert set(sd) == {"weight", "weight_scale", "bias"} and sd["weight_scale"].shape == (1, 2)
    res = b.load_state_dict(sd)
    assert not res.missing_keys and not res.unexpected_keys and torch.equal(a(x), b(x)) and b.weight.stride(0) == 208
    box = torch.nn.ModuleDict({"p": _coded_linear(dev, seed=3)})
    box.load_state_dict({f"p.{k}": v for k, v in sd.items()})
    assert torch.equal(box["p"](x), a(x))
    c = _coded_linear(dev, seed=4)
    c.load_state_dict({k: v.clone() for k, v in sd.items()}, assign=True)
    assert torch.equal(c(x), a(x)) and c.weight.stride(0) == 208 and not c.weight.requires_grad
    from axolotl_b200.models.layers import FusedLinear

    dense = FusedLinear(200, [64, 24], ["a", "b"], bias=True, dtype=a.bias.dtype, device=dev)
    with torch.no_grad():
        dense.weight.zero_()
    for target, source in ((dense, sd), (dense, {k: sd[k] for k in ("weight", "bias")}), (b, dense.state_dict()),
                           (b, {k: sd[k] for k in ("weight", "bias")}), (b, {**sd, "weight_scale": sd["weight_scale"][:, :1]})):
        before = target.weight.data.clone()
        with pytest.raises(RuntimeError, match="codes"):
            target.load_state_dict(source)
        assert torch.equal(target.weight.data, before)
    nf4 = _coded_linear(dev, 256, "nf4")
    assert set(nf4.state_dict()) == {"weight", "bias"}


@pytest.mark.gpu
@pytest.mark.parametrize("coded", [True, False])
@pytest.mark.parametrize("T", [40, 600])
def test_adapters_of_more_blocks_than_the_one_pass_kernel_takes(T, coded):
    """Nine stacked adapters: the pass over dy for t and dB at once takes eight, so they go the way of large ranks. Small integers, so that
    what the sums and the bf16 intermediates hold is exact and dB is compared bit for bit."""
    from axolotl_b200.ops.fp8 import fp8_lora_linear, quantize_fp8_weight
    from axolotl_b200.ops.lora import lora_linear

    blocks = tuple((64 * i, 64, 8 * i, 8) for i in range(9))
    K, N, R = 64, 576, 72
    g = torch.Generator().manual_seed(T)
    x, dy = (torch.randint(-1, 2, (T, n), generator=g).bfloat16() for n in (K, N))
    A, B = torch.randint(-1, 2, (R, K), generator=g).float(), torch.zeros(N, R)
    for r0, rows, c0, r in blocks:
        B[r0:r0 + rows, c0:c0 + r] = torch.randint(-1, 2, (rows, r), generator=g).float()
    Al, Bl = A.cuda().requires_grad_(True), B.cuda().requires_grad_(True)
    args = (Al, Bl, A.bfloat16().cuda(), B.bfloat16().cuda(), 1.0, blocks)
    w = torch.ones(N, K, device="cuda")
    y = fp8_lora_linear(x.cuda(), *quantize_fp8_weight(w), *args) if coded else lora_linear(x.cuda(), w.bfloat16(), *args)
    dA, dB = torch.autograd.grad(y, [Al, Bl], dy.cuda())
    low = x.double() @ A.double().t()
    for r0, rows, c0, r in blocks:
        assert torch.equal(dB[r0:r0 + rows, c0:c0 + r].cpu().double(), dy[:, r0:r0 + rows].double().t() @ low[:, c0:c0 + r])
    want = (dy.double() @ B.double()).bfloat16().double().t() @ x.double()
    assert torch.equal(dA.cpu().double(), want)


@pytest.mark.parametrize("key,name", [("unfrozen_parameters", r"mlp\.gate"), ("lora_modules_to_save", "mlp.gate"),
                                      ("unfrozen_parameters", r"layers\.\d+\.mlp\.gate")])
def test_a_router_may_be_trained_beside_codes(key, name):
    """`mlp.gate` is the router's name and the beginning of a dense layer's projection: the configuration does not know which the model has, the
    set-up does."""
    from axolotl_b200.config.load import load_cfg
    from axolotl_b200.train.run import setup_adapter

    cfg = load_cfg({**BASE, key: [name]})
    with pytest.raises(ValueError, match=r"layers\.0\.mlp\.gate_up_proj\.weight"):
        setup_adapter(cfg, _model())
    from axolotl_b200.models.config import preset
    from axolotl_b200.models.transformer import CausalLM

    moe = CausalLM(preset("tiny-qwen3-moe", num_hidden_layers=2, vocab_size=512), dtype=torch.float32, device="cpu").init_weights(0)
    setup_adapter(cfg, moe)
    trained = [n for n, p in moe.named_parameters() if p.requires_grad and "lora" not in n]
    assert trained and all(n.endswith("mlp.gate") for n in trained)
