"""A run of the serving operators together: the GPT-2-shaped block with packed weights and an MX cache, prompt chunk and single
tokens, against 64-bit arithmetic on what its buffers and cache hold."""
import math

import pytest
import torch

import mptorch_b200.quant as q
from mptorch_b200.gpt2_block import BlockConfig, QTinyGPT, ServedGPT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(5)
    cfg = BlockConfig(d_model=128, n_head=2, d_mlp=256, vocab=515, seq_len=96)
    formats = (q.QAffineFormats(), q.QSoftmaxFormats(), q.QLayerNormFormats())       # nothing rounded but weights and cache
    m = QTinyGPT(cfg, formats).cuda()
    with torch.no_grad():
        for lin in (m.block.qkv, m.block.proj, m.block.fc, m.block.out):
            lin.weight.mul_(5)
            lin.bias.normal_(std=0.1)
        m.wte.weight.mul_(20)
    return m


def dense(layer):
    """The weight that a packed layer stands for, in 64 bits: its codes are those of the quantizer on it."""
    eye = torch.eye(layer.in_features, device="cuda", dtype=torch.float32)
    plain = q.QPackedLinear.forward(layer, eye) - (0 if layer.bias is None else layer.bias)
    return plain.t().double()


def block64(served, x, kc, vc, first):
    """The block's output for rows x [T, d] at positions from ``first``, with K and V [T_all, heads, dim] as the cache holds them."""
    b, d, h = served.block, x.shape[-1], served.cfg.n_head
    w = {n: (dense(getattr(b, n)), getattr(b, n).bias.double()) for n in ("qkv", "proj", "fc", "out")}
    ln = lambda v, m: torch.nn.functional.layer_norm(v, (d,), m.weight.double(), m.bias.double(), m.eps)  # noqa: E731
    qkv = ln(x, b.ln1) @ w["qkv"][0].t() + w["qkv"][1]
    qq, k, v = (t.unflatten(-1, (h, -1)) for t in qkv.chunk(3, dim=-1))
    s = torch.einsum("thd,shd->hts", qq, kc) / math.sqrt(d // h)
    pos = first + torch.arange(x.shape[0], device="cuda")
    s = s.masked_fill(torch.arange(kc.shape[0], device="cuda") > pos[:, None], -math.inf)
    y = torch.einsum("hts,shd->thd", torch.softmax(s, -1), vc).flatten(-2)
    x = x + y @ w["proj"][0].t() + w["proj"][1]
    out = x + torch.nn.functional.gelu(ln(x, b.ln2) @ w["fc"][0].t() + w["fc"][1]) @ w["out"][0].t() + w["out"][1]
    return out, k, v


@pytest.mark.parametrize("weights", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("elem", ["e4m3", "e2m1"])
def test_served_model(model, weights, elem):
    served = ServedGPT(model, weights)
    g = torch.Generator(device="cuda").manual_seed(1)
    idx = torch.randint(0, 515, (2, 60), device="cuda", generator=g)
    cache = served.new_cache(8, 16, elem)
    pages = torch.tensor([[3, 0, 6, 1], [7, 2, 5, 4]], device="cuda", dtype=torch.int32)
    lens = torch.tensor([50, 50], device="cuda", dtype=torch.int32)
    logits = [served(idx[:, :50], cache, pages, lens)]                               # a prompt
    for t in range(50, 60):                                                          # and one token after another
        logits.append(served(idx[:, t:t + 1], cache, pages, lens + (t - 49)))
    logits = torch.cat(logits, dim=1).double()
    k, v = (t.double() for t in q.mx_cache_read(cache, pages, lens + 10, 60))
    head = dense(served.head)
    for s in range(2):
        x = served.wte(idx[s]).double() + served.wpe(torch.arange(60, device="cuda")).double()
        out, k64, v64 = block64(served, x, k[s], v[s], 0)
        # what the cache holds is within half a step of the values it was written from: 2^-4 (E4M3) or 2^-2 (E2M1) of the value, or, below
        # the format's normal numbers and above its largest one, of the block's largest; the values themselves are exact to 1e-5 of it
        rel, low = (2.0 ** -4, 2.0 ** -16) if elem == "e4m3" else (2.0 ** -2, 2.0 ** -3)
        for held, want in ((k[s], k64), (v[s], v64)):
            top = want.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1)
            over = (top / 8 if elem == "e4m3" else top / 4) * (want.abs() > 0.85 * top if elem == "e4m3" else want.abs() > 0.7 * top)
            assert ((held - want).abs() <= rel * want.abs() + (low + 1e-5) * top + over).all()
        want = out @ head.t()
        # a chain of five products, two normalisations and an attention in fp32 (each to about 1e-6 of its norm)
        assert ((logits[s] - want).norm() / want.norm()).item() < 3e-5
    # the same tokens as one chunk: the same values up to roundings that the cache makes differently
    again = served(idx, served.new_cache(8, 16, elem), pages, lens + 10).double()
    assert ((again - logits).norm() / logits.norm()).item() < 0.05


def test_generate_and_packed_layer(model):
    served = ServedGPT(model, "nvfp4")
    idx = torch.randint(0, 515, (3, 7), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    out = served.generate(idx, 9, page=8)
    assert out.shape == (3, 16) and torch.equal(out[:, :7], idx)
    assert torch.equal(served.generate(idx, 9, page=8), out)
    with pytest.raises(ValueError, match="seq_len"):
        served.generate(idx, 96)
    lin = torch.nn.Linear(64, 10).cuda()
    for fmt in ("mxfp4", "nvfp4"):
        p = q.QPackedLinear.from_linear(lin, fmt)
        x = torch.randn(4, 64, device="cuda")
        held = q.mx_quantize(lin.weight.detach(), "e2m1", 32) if fmt == "mxfp4" else q.nvfp4_quantize(lin.weight.detach())
        want = x.double() @ held.double().t() + lin.bias.double()
        assert ((p(x).double() - want).norm() / want.norm()).item() < 1e-6
        assert p(x.bfloat16()).dtype == torch.bfloat16
        r = q.QPackedLinear(torch.zeros(10, 64, device="cuda"), lin.bias, fmt)
        r.load_state_dict(p.state_dict())
        assert torch.equal(r(x), p(x))
    with pytest.raises(ValueError, match="multiple of 32"):
        q.QPackedLinear(torch.zeros(4, 40, device="cuda"))
    with pytest.raises(ValueError, match="fmt"):
        q.QPackedLinear(torch.zeros(4, 64, device="cuda"), fmt="fp8")


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.half).cuda(),
                                     lambda m: m.half().float()])
def test_packed_layer_after_conversions(fmt, convert):
    """A model's dense tensors change their type; what a packed weight stands for does not."""
    torch.manual_seed(2)
    lin = torch.nn.Linear(96, 40).cuda()
    plain = q.QPackedLinear.from_linear(lin, fmt)
    model = torch.nn.Sequential(q.QPackedLinear.from_linear(lin, fmt))
    assert convert(model) is model
    layer = model[0]
    x = torch.randn(5, 96, device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.half):
        want = plain(x.to(dtype)) - plain.bias.to(dtype) + layer.bias.to(dtype)    # the bias is a dense tensor
        got = model(x.to(dtype))
        # three roundings to the type against one of a sum that cancels
        assert got.dtype == dtype and ((got.double() - want.double()).abs() <= 4 * torch.finfo(dtype).eps * (plain(x.to(dtype)).double().abs() + plain.bias.double().abs())).all()
    if fmt == "nvfp4":
        assert layer.global_scale.dtype == torch.float32 and torch.equal(layer.global_scale, plain.global_scale)
    assert torch.equal(layer.codes, plain.codes) and torch.equal(layer.scales, plain.scales)
