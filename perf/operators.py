"""The 8-bit block operators as measurable cases: E4M3 codes with a power-of-two scale for each row and 128 columns of an
activation, and an fp32 scale for each 128 x 128 block of a frozen weight.

* ``linear``: ``y = x8 W8^T``, a frozen projection in a generation step or an evaluation pass;
* ``frozen``: the same with its input gradient ``dx = dy8 W8`` (the projections without an adapter, in training);
* ``lora``: a projection with an adapter in training, forward and backward: ``y = x8 W8^T + (s x A^T) B^T``,
  ``dx = dy8 W8 + (s dy B) A``, ``dA = (s dy B)^T x8`` from the saved 8-bit rows, ``dB = dy^T (s x A^T)``;
* ``checkpoint``: a layer input put into the 8-bit store in the forward pass and taken back in the backward pass.

``x8`` is ``x`` at its 8-bit values: ``q s`` with ``s = 2^ceil(log2(max |x| / 448))`` of the block (1 for a block of zeros) and ``q``
the nearest E4M3 number to ``x / s``, ties to even. Sizes are those of the models of ``perf/cases.py``."""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128
RANK, ALPHA = 16, 32


def listed():
    return [
        # one chat user: a token through the attention output projection of the 8B model (the smallest call, latency counts)
        dict(name="linear_one_token", kind="linear", tokens=1, k=4096, n=4096),
        # a small evaluation batch through gate | up of the small model
        dict(name="linear_24_tokens_1b", kind="linear", tokens=24, k=2048, n=11264),
        # a rollout batch of reinforcement learning through the down projection
        dict(name="linear_64_tokens", kind="linear", tokens=64, k=14336, n=4096),
        # the packed prompts of such a batch, an odd number of tokens, through q | k | v
        dict(name="linear_prompts", kind="linear", tokens=777, k=4096, n=6144),
        # gate | up of the headline row: 8192 packed tokens (the largest)
        dict(name="linear_packed_row", kind="linear", tokens=8192, k=4096, n=28672),
        # a frozen projection of the small model in training, widths that end inside a block
        dict(name="frozen_ragged", kind="frozen", tokens=1531, k=2008, n=2904),
        # the output projection without an adapter, packed row
        dict(name="frozen_packed_row", kind="frozen", tokens=8192, k=4096, n=4096),
        # a short fine-tuning row through q | k | v
        dict(name="lora_short_row", kind="lora", tokens=960, k=4096, n=6144),
        # the headline row through the down projection
        dict(name="lora_packed_row", kind="lora", tokens=8192, k=14336, n=4096),
        # the layer input of a short row of the small model
        dict(name="checkpoint_short_row", kind="checkpoint", tokens=960, k=2048),
        # an odd number of tokens and a width that ends inside a block
        dict(name="checkpoint_ragged", kind="checkpoint", tokens=5003, k=4072),
        # the headline row over four micro-batches of one layer
        dict(name="checkpoint_packed_rows", kind="checkpoint", tokens=32768, k=4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "frozen", "lora", "checkpoint"])
    if kind == "checkpoint":
        return dict(kind=kind, tokens=_log(rng, 64, 32768), k=8 * _log(rng, 64, 512))
    while True:
        tokens = _log(rng, 1 if kind == "linear" else 64, 8192)
        k, n = 8 * _log(rng, 64, 1792), 8 * _log(rng, 64, 3584)
        if tokens * k * n <= 8192 * 4096 * (28672 if kind == "linear" else 14336):
            return dict(kind=kind, tokens=tokens, k=k, n=n)


def _activations(tokens, k, g):
    """Hidden states: a few channels carry values far above the others'."""
    wide = 1 + 12 * (torch.rand(k, device=DEV, generator=g) < 0.01).float()
    return (torch.randn(tokens, k, device=DEV, generator=g) * wide).bfloat16()


def _weight(n, k, g):
    """A frozen projection as block-FP8 checkpoints hold it: codes [n, k], scales [ceil(n / 128), ceil(k / 128)]. Rows of codes start on
    16 bytes, as a program lays them out once for bulk tensor copies."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(nb * BLOCK, kb * BLOCK, device=DEV)
    w[:n, :k] = torch.randn(n, k, device=DEV, generator=g) * k ** -0.5
    blocks = w.view(nb, BLOCK, kb, BLOCK)
    scale = blocks.abs().amax((1, 3)) / 448
    codes = (blocks / scale[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:n, :-(-k // 16) * 16].to(torch.float8_e4m3fn).contiguous()
    return codes[:, :k], scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t, k = case["tokens"], case["k"]
    s = {"kind": case["kind"], "x": _activations(t, k, g)}
    if case["kind"] == "checkpoint":
        return s
    n = case["n"]
    s["codes"], s["scale"] = _weight(n, k, g)
    if case["kind"] == "linear":
        return s
    # the loss leaves out the prompts: their gradient rows are zero
    answer = torch.rand(t, 1, device=DEV, generator=g) < 0.7
    s["dy"] = (torch.randn(t, n, device=DEV, generator=g) * 1e-3 * answer).bfloat16()
    if case["kind"] == "lora":
        s["A"] = ((torch.rand(RANK, k, device=DEV, generator=g) * 2 - 1) * k ** -0.5).bfloat16()
        s["B"] = (torch.randn(n, RANK, device=DEV, generator=g) * 0.02).bfloat16()
    return s


def _rows8(x):
    """``x`` at its 8-bit values, in 32 bits."""
    t, k = x.shape
    kb = -(-k // BLOCK)
    pad = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k)).view(t, kb, BLOCK)
    top = pad.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top / 448)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), (e - (m == 0.5).int()).clamp(min=-126)), torch.ones_like(top))
    return ((pad / scale).to(torch.float8_e4m3fn).float() * scale).view(t, kb * BLOCK)[:, :k]


def _weight8(codes, scale):
    n, k = codes.shape
    return codes.float() * scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def _plain(s):
    x, kind = s["x"], s["kind"]
    if kind == "checkpoint":
        return _rows8(x).to(x.dtype)
    w = _weight8(s["codes"], s["scale"])
    x8 = _rows8(x)
    y = x8 @ w.t()
    if kind == "linear":
        return y.bfloat16()
    dy = s["dy"]
    dx = _rows8(dy) @ w
    if kind == "frozen":
        return {"y": y.bfloat16(), "dx": dx.bfloat16()}
    a, b, c = s["A"].float(), s["B"].float(), ALPHA / RANK
    low, tall = c * (x.float() @ a.t()), c * (dy.float() @ b)
    return {"y": (y + low @ b.t()).bfloat16(), "dx": (dx + tall @ a).bfloat16(), "dA": (tall.t() @ x8).bfloat16(),
            "dB": (dy.float().t() @ low).bfloat16()}


def run(s):
    if not own:
        with torch.no_grad():
            return _plain(s)
    from axolotl_b200.ops.fp8 import fp8_linear, fp8_lora_linear
    from axolotl_b200.train.activation_memory import make_store

    x, kind = s["x"], s["kind"]
    if kind == "checkpoint":
        store = make_store("fp8", x.device)
        return store.get(store.put(x))
    if kind == "linear":
        with torch.no_grad():
            return fp8_linear(x, s["codes"], s["scale"])
    x = x.detach().requires_grad_(True)
    if kind == "frozen":
        y = fp8_linear(x, s["codes"], s["scale"])
        (dx,) = torch.autograd.grad(y, [x], s["dy"])
        return {"y": y, "dx": dx}
    a, b = s["A"].detach().requires_grad_(True), s["B"].detach().requires_grad_(True)
    n = s["codes"].shape[0]
    y = fp8_lora_linear(x, s["codes"], s["scale"], a, b, s["A"], s["B"], ALPHA / RANK, ((0, n, 0, RANK),))
    dx, da, db = torch.autograd.grad(y, [x, a, b], s["dy"])
    return {"y": y, "dx": dx, "dA": da, "dB": db}


def work(case):
    t, k = case["tokens"], case["k"]
    rows = t * k + 4 * t * -(-k // BLOCK)                       # 8-bit codes and their scales
    if case["kind"] == "checkpoint":
        return {"bytes": 4 * t * k + 2 * rows, "flops": 0}
    n = case["n"]
    weight = n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK)
    if case["kind"] == "linear":
        return {"bytes": 2 * t * (k + n) + weight, "flops": 2 * t * n * k}
    if case["kind"] == "frozen":
        return {"bytes": 4 * t * (k + n) + weight, "flops": 4 * t * n * k}
    return {"bytes": 4 * t * (k + n) + weight + 4 * RANK * (k + n), "flops": 4 * t * n * k + 6 * t * RANK * (n + k)}


def _exact_rows8(x):
    """The definition in 64 bits: the nearest multiple of the step that E4M3 has at that magnitude (2^-9 below 2^-6)."""
    t, k = x.shape
    out = torch.empty(t, k, dtype=torch.float64, device=x.device)
    for c in range(0, k, BLOCK):
        v = x[:, c:c + BLOCK].double()
        top = v.abs().amax(1, keepdim=True)
        scale = torch.where(top > 0, torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300)) - math.log2(448) - 1e-12).clamp(min=-126)), 1.0)
        u = v / scale
        step = torch.exp2(torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6))) - 3)
        out[:, c:c + BLOCK] = torch.round(u / step) * step * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    x, kind = s["x"], case["kind"]
    x8 = _exact_rows8(x)
    if kind == "checkpoint":
        return x8
    n, k = s["codes"].shape
    rows, cols = (torch.arange(m, device=DEV) // BLOCK for m in (n, k))
    w = s["codes"].double() * s["scale"].double()[rows][:, cols]
    y = torch.einsum("tk,nk->tn", x8, w)
    if kind == "linear":
        return y
    dy = s["dy"].double()
    dx = torch.einsum("tn,nk->tk", _exact_rows8(s["dy"]), w)
    if kind == "frozen":
        return {"y": y, "dx": dx}
    a, b, c = s["A"].double(), s["B"].double(), ALPHA / RANK
    low, tall = torch.einsum("tk,rk->tr", x.double(), a) * c, torch.einsum("tn,nr->tr", dy, b) * c
    y += torch.einsum("tr,nr->tn", low, b)
    dx += torch.einsum("tr,rk->tk", tall, a)
    return {"y": y, "dx": dx, "dA": torch.einsum("tr,tk->rk", tall, x8), "dB": torch.einsum("tn,tr->nr", dy, low)}
