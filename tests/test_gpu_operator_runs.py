"""The RMS norm, the gated block and the 8-bit product as a program uses them together: a block's forward and backward pass against
the formulas in 64 bits, an 8-bit forward pass, both captured into graphs and replayed, on streams of their own, and two at once."""
import pytest
import torch

from gpu_util import check, library, rel, stream, sync

pytestmark = pytest.mark.gpu

BF16, F8 = torch.bfloat16, torch.float8_e4m3fn
EPS = 1e-6


class Block:
    """y = h + down(silu(gate(n)) up(n)), n = norm(h), h = x + r, with the weights' transposed copies, and its gradients."""

    def __init__(self, M, D, F, seed):
        g = torch.Generator().manual_seed(seed)
        make = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).to(BF16).cuda()  # noqa: E731
        self.M, self.D, self.F = M, D, F
        self.x, self.r, self.dy = make(M, D), make(M, D), make(M, D)
        self.w, self.down = make(2 * F, D, scale=D ** -0.5), make(D, F, scale=F ** -0.5)
        self.w_t, self.down_t = self.w.t().contiguous(), self.down.t().contiguous()
        self.gamma = (1 + 0.1 * torch.randn(D, generator=g)).cuda()
        bits = self.gamma.view(torch.int32)
        self.hi, self.lo = (bits >> 16).to(torch.int16), (bits & 0xffff).to(torch.int16)
        empty = lambda *shape, dtype=BF16: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
        self.h, self.n, self.a, self.gu, self.y = empty(M, D), empty(M, D), empty(M, F), empty(M, 2 * F), empty(M, D)
        self.dgu, self.dn, self.dx = empty(M, 2 * F), empty(M, D), empty(M, D)
        self.dw, self.ddown, self.dgamma = (empty(*s, dtype=torch.float32) for s in ((2 * F, D), (D, F), (D,)))
        lib = library()
        need = max(lib.tgk_rmsnorm_bwd_workspace(M, D), lib.tgk_gemm_wgrad_workspace(M, 2 * F, D), lib.tgk_gemm_wgrad_workspace(M, D, F), 16)
        self.workspace = empty(need, dtype=torch.uint8)

    def step(self):
        lib, st, M, D, F = library(), stream(), self.M, self.D, self.F
        p = {k: v.data_ptr() for k, v in vars(self).items() if torch.is_tensor(v)}
        ws, size = p["workspace"], self.workspace.numel()
        check(lib.tgk_rmsnorm_fwd(st, M, D, p["x"], p["r"], p["hi"], p["lo"], p["h"], p["n"], None, None, 0, EPS))
        check(lib.tgk_gated_fwd(st, M, F, D, p["n"], D, p["w"], D, p["a"], F, p["gu"], 2 * F, 0))
        check(lib.tgk_gemm_fwd(st, M, D, F, p["a"], F, p["down"], F, p["y"], D, p["h"], D, None, 0))
        check(lib.tgk_gated_bwd(st, M, F, D, p["dy"], D, p["down_t"], D, p["gu"], 2 * F, p["dgu"], 2 * F, p["w_t"], 2 * F, p["dn"], D, 0))
        check(lib.tgk_gemm_wgrad(st, M, 2 * F, D, p["dgu"], 2 * F, p["n"], D, p["dw"], D, 0, ws, size))
        check(lib.tgk_gemm_wgrad(st, M, D, F, p["dy"], D, p["a"], F, p["ddown"], F, 0, ws, size))
        check(lib.tgk_rmsnorm_bwd(st, M, D, p["h"], p["dn"], p["hi"], p["lo"], p["dy"], p["dx"], p["dgamma"], EPS, 0, ws, size))

    OUTPUTS = ("y", "dx", "dw", "ddown", "dgamma")

    def outputs(self):
        return [getattr(self, name).clone() for name in self.OUTPUTS]

    def clear(self):
        for name in self.OUTPUTS:
            getattr(self, name).zero_()

    def exact(self):
        """In 64 bits on the CPU, from the operators' inputs; gradients by automatic differentiation."""
        wide = lambda t: t.double().cpu().requires_grad_()  # noqa: E731
        h = wide((self.x.float() + self.r.float()).to(BF16))
        gamma, w, down = wide(self.gamma), wide(self.w), wide(self.down)
        n = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * gamma
        both = n @ w.t()
        y = h + (torch.nn.functional.silu(both[:, :self.F]) * both[:, self.F:]) @ down.t()
        y.backward(self.dy.double().cpu())
        return [y.detach(), h.grad, w.grad, down.grad, gamma.grad]


# Every output is a chain of at most eight values rounded to bfloat16, each off by 2^-8 at most and in no common direction; the sum of all
# in one is the bound: 8 x 2^-8.
CHAIN = 8 * 2.0 ** -8


@pytest.mark.parametrize("M,D,F", [(128, 128, 256), (384, 256, 640), (1024, 768, 2048)])
def test_a_block_and_its_gradients(M, D, F):
    block = Block(M, D, F, M)
    block.step()
    sync()
    for name, got, want in zip(block.OUTPUTS, block.outputs(), block.exact()):
        assert rel(got.float().cpu().numpy(), want.numpy()) <= CHAIN, name


def test_a_block_captured_and_replayed_between_eager_steps():
    block, other = Block(256, 256, 512, 7), Block(256, 256, 512, 8)
    block.step(), other.step()
    sync()
    want, want_other = block.outputs(), other.outputs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block.step()
    for _ in range(4):
        block.clear(), other.clear()
        graph.replay()
        other.step()
        sync()
        assert all(torch.equal(a, b) for a, b in zip(block.outputs(), want))
        assert all(torch.equal(a, b) for a, b in zip(other.outputs(), want_other))


def test_two_blocks_on_streams_of_their_own():
    blocks = [Block(512, 256, 1024, s) for s in (1, 2)]
    want = []
    for block in blocks:
        block.step()
        sync()
        want.append(block.outputs())
        block.clear()
    streams = [torch.cuda.Stream() for _ in blocks]
    sync()
    for _ in range(5):
        for block, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                block.step()
    sync()
    for block, values in zip(blocks, want):
        assert all(torch.equal(a, b) for a, b in zip(block.outputs(), values))


class Forward8:
    """An 8-bit forward pass of the block: the norm leaves codes for the first projection; its gated result is quantised for the second."""

    def __init__(self, M, D, F, seed):
        block = self.block = Block(M, D, F, seed)
        codes = lambda *shape: torch.empty(*shape, dtype=torch.uint8, device="cuda")  # noqa: E731
        groups = lambda n: -(-n // 128)  # noqa: E731
        self.n8, self.n_scales = codes(M, D), torch.empty(groups(D), M, device="cuda")
        self.a8, self.a_scales = codes(M, F), torch.empty(groups(F), M, device="cuda")
        self.down8, self.down_scales = codes(D, F), torch.empty(groups(D), groups(F), device="cuda")
        self.proj, self.proj8, self.proj_scales = block.w[:D].contiguous(), codes(D, D), torch.empty(groups(D), groups(D), device="cuda")
        self.p = torch.empty(M, D, dtype=BF16, device="cuda")
        lib = library()
        check(lib.tgk_quantize_tiles(stream(), D, F, block.down.data_ptr(), F, self.down8.data_ptr(), F, self.down_scales.data_ptr(), groups(F)))
        check(lib.tgk_quantize_tiles(stream(), D, D, self.proj.data_ptr(), D, self.proj8.data_ptr(), D, self.proj_scales.data_ptr(), groups(D)))

    def step(self):
        lib, st, b = library(), stream(), self.block
        M, D, F = b.M, b.D, b.F
        check(lib.tgk_rmsnorm_fwd(st, M, D, b.x.data_ptr(), b.r.data_ptr(), b.hi.data_ptr(), b.lo.data_ptr(), b.h.data_ptr(), b.n.data_ptr(), self.n8.data_ptr(),
                                  self.n_scales.data_ptr(), M, EPS))
        check(lib.tgk_gemm_q8(st, M, D, D, self.n8.data_ptr(), D, self.n_scales.data_ptr(), M, self.proj8.data_ptr(), D, self.proj_scales.data_ptr(),
                              self.proj_scales.shape[1], self.p.data_ptr(), D, None, 0))
        check(lib.tgk_gated_fwd(st, M, F, D, b.n.data_ptr(), D, b.w.data_ptr(), D, b.a.data_ptr(), F, None, 0, 0))
        check(lib.tgk_quantize_rows(st, M, F, b.a.data_ptr(), F, self.a8.data_ptr(), F, self.a_scales.data_ptr(), M))
        check(lib.tgk_gemm_q8(st, M, D, F, self.a8.data_ptr(), F, self.a_scales.data_ptr(), M, self.down8.data_ptr(), F, self.down_scales.data_ptr(),
                              self.down_scales.shape[1], b.y.data_ptr(), D, b.h.data_ptr(), D))


@pytest.mark.parametrize("M,D,F", [(1, 128, 256), (33, 272, 528), (300, 640, 1712)])
def test_an_eight_bit_forward_pass(M, D, F):
    """Both operands of a product are off by 2^-4 at most through their codes, everything else by a few 2^-8: 2 x 2^-4 + 8 x 2^-8."""
    f = Forward8(M, D, F, M + D)
    f.step()
    sync()
    b = f.block
    y = b.exact()[0]
    assert rel((b.y.float() - b.h.float()).cpu().numpy(), (y - b.h.double().cpu()).numpy()) <= 2 * 2.0 ** -4 + CHAIN
    n = b.h.double()
    n = n / torch.sqrt(n.square().mean(1, keepdim=True) + EPS) * b.gamma.double()
    assert rel(f.p.float().cpu().numpy(), (n @ f.proj.double().t()).cpu().numpy()) <= 2 * 2.0 ** -4 + CHAIN


def test_an_eight_bit_forward_pass_captured_and_replayed():
    f = Forward8(65, 256, 512, 3)
    f.step()
    sync()
    want = [f.block.y.clone(), f.p.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f.step()
    for i in range(4):
        f.block.y.zero_(), f.p.zero_(), f.a8.zero_(), f.n_scales.zero_()
        graph.replay()
        sync()
        assert torch.equal(f.block.y, want[0]) and torch.equal(f.p, want[1])
        new = Forward8(65, 256, 512, 100 + i)  # other inputs in the captured buffers: no replay keeps an answer
        f.block.x.copy_(new.block.x)
        graph.replay()
        sync()
        changed = f.block.y.clone()
        f.step()
        sync()
        assert torch.equal(f.block.y, changed) and not torch.equal(changed, want[0])
        want = [changed, f.p.clone()]
