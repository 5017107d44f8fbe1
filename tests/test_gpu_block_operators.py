"""4-bit Linears, norms over the residual and rotary positions as a block uses them together: a run of all of them, recorded, on other streams, in a
module and in the encoder, over more memory than 32 bits address, and into memory that is an input's."""

import pytest
import torch

from test_gpu_linear_i4 import _check as check_linear, _operands
from test_gpu_norm_residual import _close, _inputs, _reference
from test_gpu_rotary import _check as check_rotary, _frequencies

pytestmark = pytest.mark.gpu


def _weights(N, K, group, dtype, g):
    w = torch.randn((N, K), generator=g, device="cuda") * K ** -0.5
    from samfast_amd import quantize_weight_int4
    return (*quantize_weight_int4(w, group, True, dtype), 0.02 * torch.randn((N,), generator=g, device="cuda"))


class _Block:
    """One pre-norm attention half of a block over 14 x 14 windows, with a gate and a norm behind the branch."""

    def __init__(self, C, nH, dtype, stream):
        from samfast_amd import grid_positions, rotary_frequencies
        g = torch.Generator(device="cuda").manual_seed(C)
        self.nH, self.hd, self.dtype, self.stream = nH, C // nH, dtype, stream
        self.qkv, self.proj = _weights(3 * C, C, 64, dtype, g), _weights(C, C, 128, dtype, g)
        self.post, self.pre = (((1 + 0.1 * torch.randn(C, generator=g, device="cuda")).to(dtype), None, 1e-6) for _ in range(2))
        self.positions = grid_positions(14, 14, device="cuda")
        self.frequencies = rotary_frequencies(self.hd // 4, device="cuda").expand(2, -1).contiguous()
        self.tables = torch.zeros((27, self.hd), dtype=dtype, device="cuda")

    def linear(self, x, w, group):
        from samfast_amd import ops
        return ops.linear_i4(x, w[0], w[1], w[2], w[3], group_size=group)

    def __call__(self, tokens, residual, gate):
        from samfast_amd import ops
        B, T, C = tokens.shape
        qkv = self.linear(tokens, self.qkv, 64)
        q, k, v = qkv.view(B, T, 3, self.nH, self.hd).permute(2, 0, 3, 1, 4)
        qr, kr = ops.rotary(q, k, self.positions, self.frequencies, interleaved=True)
        heads = ops.attn_relpos(qr, kr, v, self.tables, self.tables, (14, 14))
        branch = self.linear(heads.permute(0, 2, 1, 3).reshape(B, T, C), self.proj, 128)
        total, normed = ops.norm_residual(branch, residual, gate=gate, post=self.post, pre=self.pre, rms=True)
        return dict(qkv=qkv, q=q, k=k, v=v, qr=qr, kr=kr, heads=heads, branch=branch, total=total, normed=normed)


@pytest.mark.parametrize("dtype,stream", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_a_block_s_run(dtype, stream):
    block = _Block(256, 4, dtype, stream)
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    tokens, residual, gate = r(3, 196, 256).to(dtype), r(3, 196, 256).to(stream), r(3, 256).to(dtype)
    o = block(tokens, residual, gate)
    # every step against its formula, on what the step before it gave
    check_linear(o["qkv"], tokens, *block.qkv, 64)
    for turned, plain in ((o["qr"], o["q"]), (o["kr"], o["k"])):
        check_rotary(turned, plain, block.positions, block.frequencies, True, 1.0)
    p = torch.softmax(o["qr"].double() @ o["kr"].double().transpose(-1, -2).contiguous() * block.hd ** -0.5, -1)
    assert (o["heads"].double() - p @ o["v"].double().contiguous()).abs().max() <= 2e-2
    check_linear(o["branch"], o["heads"].permute(0, 2, 1, 3).reshape(3, 196, 256), *block.proj, 128)
    flat = lambda t: t.reshape(-1, 256)
    total, normed = _reference(flat(o["branch"]), flat(residual), gate, block.post, block.pre, True, 1.0, 1.0)
    _close(flat(o["total"]), total, 256 * 2.0 ** -24)
    spread = (total.abs().amax(-1) / (total.square().mean(-1) + 1e-6).sqrt()).max()
    _close(flat(o["normed"]), normed, 256 * 2.0 ** -24 * float(spread))


def test_a_recorded_run_replays_with_new_inputs():
    block = _Block(256, 4, torch.bfloat16, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(4)
    draw = lambda: (torch.randn((2, 196, 256), generator=g, device="cuda").bfloat16(), torch.randn((2, 196, 256), generator=g, device="cuda"),
                    torch.randn((2, 256), generator=g, device="cuda").bfloat16())
    held = draw()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(*held)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two recordings of the same tensors
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(*held)
        graphs.append((graph, out))
    for step in range(4):
        fresh = draw()
        want = block(*fresh)
        for h, f in zip(held, fresh):
            h.copy_(f)
        graph, out = graphs[step % 2]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[name], want[name]) for name in want)


@pytest.mark.parametrize("M,K,N", [(700, 1000, 1003), (64, 4096, 1024), (4096, 1280, 5120)])  # one tile each, K split, the weights written out
def test_recorded_linears_with_workspaces_on_two_streams(M, K, N):
    from samfast_amd import _lib, ops
    need = _lib.load().samfast_linear_i4_workspace(M, N, K)
    assert (need > 0) == (M != 700)
    sets = [_operands(M, K, N, 64, True, torch.bfloat16, seed=s) for s in range(2)]
    want = [ops.linear_i4(*s, group_size=64) for s in sets]
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_i4(*s, group_size=64)
        graphs.append((graph, out, torch.cuda.Stream()))
    for _ in range(5):
        for graph, out, stream in graphs:
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [ops.linear_i4(*s, group_size=64) for s in sets]  # beside them
        torch.cuda.synchronize()
        for w, e, (_, out, _) in zip(want, eager, graphs):
            assert torch.equal(out, w) and torch.equal(e, w)
            out.zero_()


def test_on_another_stream():
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(100, 512, 300, 32, True, torch.float16)
    nx, residual, gate, (post, pre) = _inputs(64, 300, torch.float16, torch.float16, 2)
    q = torch.randn((2, 3, 40, 64), device="cuda").half()
    positions, freq = torch.arange(40, device="cuda"), _frequencies(16, 1)
    run = lambda: (ops.linear_i4(x, codes, scales, z, b, group_size=32), *ops.norm_residual(nx, residual, gate=gate, post=post, pre=pre), ops.rotary(q, None, positions, freq)[0])
    want = run()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = run()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M", [1, 50, 600])
@pytest.mark.parametrize("zero_points", [False, True])
def test_module(M, zero_points):
    from samfast_amd import Int4Linear
    torch.manual_seed(M)
    linear = torch.nn.Linear(200, 72).requires_grad_(False)
    for dtype in (torch.bfloat16, torch.float16):
        module = Int4Linear.from_float(linear, 64, zero_points).to("cuda", dtype)
        x = torch.randn((2, M, 200), device="cuda").to(dtype)
        check_linear(module(x), x, module.codes, module.scales, module.zeros, module.bias, 64)
        assert torch.equal(module(x.float()), module(x).float())


def test_encoder_with_4_bit_linears():
    """The swap in an image encoder: the same tokens as with the dequantised weights in half-type Linears, to what rounding those leaves."""
    from samfast_amd import apply_int4_weights
    from samfast_amd.modeling.image_encoder import ImageEncoderViT
    torch.manual_seed(0)
    encoder = ImageEncoderViT(img_size=1024, embed_dim=256, depth=2, num_heads=4, use_rel_pos=True, window_size=14, global_attn_indexes=(1,)).requires_grad_(False).eval()
    encoder.to("cuda", torch.bfloat16)
    plain = ImageEncoderViT(img_size=1024, embed_dim=256, depth=2, num_heads=4, use_rel_pos=True, window_size=14, global_attn_indexes=(1,)).requires_grad_(False).eval()
    plain.to("cuda", torch.bfloat16).load_state_dict(encoder.state_dict())
    apply_int4_weights(encoder, group_size=64)
    for name, module in encoder.named_modules():
        if type(module).__name__ == "Int4Linear":
            plain.get_submodule(name).weight.copy_(module.weight)
    x = torch.randn((1, 3, 1024, 1024), device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        got, want = encoder(x).float(), plain(x).float()
    cos = torch.nn.functional.cosine_similarity(got.flatten(), want.flatten(), 0)
    assert torch.isfinite(got).all() and cos >= 0.999


@pytest.mark.parametrize("N", [8192, 1029])  # the weights written out, and tiles
def test_linear_beyond_32_bits(N):
    from samfast_amd import ops
    M, K = 290000, 8192  # 4.75e9 bytes of x, and of y at 8192 outputs
    _, codes, scales, z, b = _operands(1, K, N, 128, True, torch.bfloat16)
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 131071, 131072, 262143, 262144, 262145, M - 130, M - 2, M - 1], device="cuda")
    x[at] = torch.randn((len(at), K), device="cuda").bfloat16()
    y = ops.linear_i4(x, codes, scales, z, b, group_size=128)
    check_linear(y[at].contiguous(), x[at].contiguous(), codes, scales, z, b, 128)
    assert torch.equal(y[M // 2], b.bfloat16()) and torch.equal(y[M - 3], b.bfloat16())


def test_rows_and_heads_beyond_32_bits():
    from samfast_amd import ops
    M, K = 290000, 8192
    x = torch.randn((K,), device="cuda").bfloat16().expand(M, K).contiguous()
    _, _, _, (post, pre) = _inputs(1, K, torch.bfloat16, torch.bfloat16, 0)
    x[M - 1] = torch.randn((K,), device="cuda").bfloat16()
    total, normed = ops.norm_residual(x, x, post=post, pre=pre)
    for row in (0, 131072, 262144, M - 2, M - 1):
        one = ops.norm_residual(x[row:row + 1], x[row:row + 1], post=post, pre=pre)
        assert torch.equal(total[row], one[0][0]) and torch.equal(normed[row], one[1][0])
    del total, normed
    heads = x.view(1, M, 64, 128).permute(0, 2, 1, 3)
    positions, freq = torch.arange(M, device="cuda") + (1 << 20), _frequencies(64, 1)
    turned = ops.rotary(heads, None, positions, freq)[0]
    for token in (0, 131072, 262144, M - 1):
        check_rotary(turned[:, :, token:token + 1], heads[:, :, token:token + 1], positions[token:token + 1], freq, False, 1.0)



def test_outs_that_would_be_read_after_they_are_written_are_refused():
    from samfast_amd import ops
    q, k = (torch.randn((2, 4, 10, 64), device="cuda").bfloat16() for _ in range(2))
    positions, freq = torch.arange(10, device="cuda"), _frequencies(32, 1)
    memory = torch.zeros(2 * 4 * 10 * 64 + 64, dtype=torch.bfloat16, device="cuda")
    shifted = memory[64:].view(2, 4, 10, 64)
    source = memory[:-64].view(2, 4, 10, 64)
    one_token = torch.zeros((2, 4, 1, 64), dtype=q.dtype, device="cuda").expand(2, 4, 10, 64)
    for args, out in [((q, k), (k, q)), ((source, None), (shifted, None)), ((q, k), (q, one_token)),
                      ((q, q.transpose(0, 1).reshape(2, 4, 10, 64)), (q.view(4, 2, 10, 64).transpose(0, 1), k))]:
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.rotary(*args, positions, freq, out=out)
    same = torch.empty_like(q)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.rotary(q, k, positions, freq, out=(same, same))
    want = ops.rotary(q, k, positions, freq)
    got = ops.rotary(q, k, positions, freq, out=(torch.empty_like(q), k))
    assert torch.equal(got[0], want[0]) and torch.equal(k, want[1])

    x, residual, gate, (post, pre) = _inputs(8, 64, torch.bfloat16, torch.bfloat16, 2)
    memory = torch.zeros(8 * 64 + 64, dtype=torch.bfloat16, device="cuda")
    memory[:512] = residual.flatten()
    for args, out in [(dict(residual=memory[:512].view(8, 64)), memory[64:].view(8, 64)), (dict(gate=memory[:128].view(2, 64)), memory[:512].view(8, 64)),
                      (dict(x=memory[:512].view(8, 64)), memory[8:520].view(8, 64))]:
        with pytest.raises(RuntimeError, match="overlaps"):
            ops.norm_residual(**dict(dict(x=x, residual=residual, gate=gate, post=post, pre=pre), **args), out=out)
    want = ops.norm_residual(x, residual, gate=gate, post=post, pre=pre)
    into = x.clone()
    got = ops.norm_residual(into, residual, gate=gate, post=post, pre=pre, out=into)
    assert torch.equal(into, want[0]) and torch.equal(got[1], want[1])


def test_recorded_linear_with_copied_rows():
    """Rows of 1288 values: their copies lie in the recording's own memory, and are made again at each replay."""
    from samfast_amd import ops
    x, codes, scales, z, b = _operands(5000, 1288, 3001, 64, True, torch.bfloat16)
    call = lambda: ops.linear_i4(x, codes, scales, z, b, group_size=64)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_copied_rows_beyond_32_bits():
    from samfast_amd import ops
    M, K, N = 290000, 8200, 1029  # 4.76e9 bytes of x, and as many of its copies
    _, codes, scales, z, b = _operands(1, K, N, 128, True, torch.bfloat16)
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 130943, 130944, 261888, 262144, M - 130, M - 2, M - 1], device="cuda")
    x[at] = torch.randn((len(at), K), device="cuda").bfloat16()
    y = ops.linear_i4(x, codes, scales, z, b, group_size=128)
    check_linear(y[at].contiguous(), x[at].contiguous(), codes, scales, z, b, 128)
    assert torch.equal(y[M // 2], b.bfloat16()) and torch.equal(y[M - 3], b.bfloat16())


def test_tiles_beyond_32_bits():
    from samfast_amd import _lib, ops
    M, K, N = 290000, 8192, 100
    assert _lib.load().samfast_linear_i4_workspace(M, N, K) == 0  # tiles
    _, codes, scales, z, b = _operands(1, K, N, 128, True, torch.bfloat16)
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 131071, 131072, 262143, 262144, M - 1], device="cuda")
    x[at] = torch.randn((len(at), K), device="cuda").bfloat16()
    y = ops.linear_i4(x, codes, scales, z, b, group_size=128)
    check_linear(y[at].contiguous(), x[at].contiguous(), codes, scales, z, b, 128)
    assert torch.equal(y[M // 2], b.bfloat16())


def test_module_in_an_fp32_model():
    from samfast_amd import Int4Linear
    torch.manual_seed(0)
    module = Int4Linear.from_float(torch.nn.Linear(200, 72).requires_grad_(False), 64, True).to("cuda")
    x = torch.randn((2, 5, 200), device="cuda")
    want = module(x)
    for cast in (module.float, module.double):
        got = cast()(x)
        assert got.dtype == torch.float32 and torch.equal(got, want)
    half = x.bfloat16()
    check_linear(module(half), half, module.codes, module.scales, module.zeros, module.bias, 64)
