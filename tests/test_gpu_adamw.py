"""AdamW kernels (`ops.adamw_step`, `ops.adamw_read8`) against the definition in 64 bits, and against the host's loops to the bit."""
import pytest
import torch

import bagua_core_b200.ops as ops
import test_cpu_adamw as host

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtypes", host.TYPES)
@pytest.mark.parametrize("t", [1, 1000])
def test_step_with_fp32_moments(dtypes, t):
    host.check_step32("cuda", dtypes, t)


@pytest.mark.parametrize("dtypes", host.TYPES)
def test_step_with_8_bit_moments(dtypes):
    host.check_step8("cuda", dtypes, 3)


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_tensors_that_start_anywhere(offset):
    host.check_step8("cuda", (torch.float32, torch.bfloat16), 3, offset=offset)


def test_8_bit_moments_follow_their_mean():
    host.check_mean("cuda")


def test_special_values():
    host.check_special("cuda")


def test_fp32_moments_that_start_anywhere():
    host.check_unaligned32("cuda")


def test_graphs_notice_a_step():
    host.check_versions("cuda")


def test_8_bit_moments_in_another_order():
    host.check_other_orders("cuda")


def test_weight_decay_is_taken_as_it_is():
    host.check_weight_decay("cuda")


def test_graphs_notice_all_that_is_written():
    host.check_versions_of_all_written("cuda")


def test_refusals():
    host.check_refusals("cuda")


def test_step_number_in_a_tensor():
    host.check_step_on_device("cuda")


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count,size", [(1, 300_001), (45, 777), (401, 130)])
def test_host_and_gpu_give_the_same_bits(bits, count, size):
    """... of the moments; with those in 8 bits the GPU's square root and reciprocal are its approximate ones, within 2^-22 each, which may
    move a parameter by a rounding: half a step of fp32 at each of three steps, and 2^-21 of updates of at most 10 lr."""
    got = []
    for device in ("cpu", "cuda"):
        ps, gs, ms, vs = host.tensors([size] * count, (torch.float32, torch.float32), device)
        cs = [torch.zeros_like(p, dtype=torch.bfloat16) for p in ps]
        more, ss = {}, []
        if bits == 8:
            state = [ops.adamw_state8(p) for p in ps]
            ms, vs, ss = ([s[i] for s in state] for i in range(3))
            more = dict(scales=ss, seed=11)
        for t in (1, 2, 3):
            ops.adamw_step(ps, gs, ms, vs, step=t, copies=cs, **host.HYPER, **more)
        got.append([[x.cpu() for x in ms + vs + ss], [p.cpu() for p in ps], [c.cpu() for c in cs]])
    assert all(torch.equal(a, b) for a, b in zip(got[0][0], got[1][0]))
    for (p, c), (q, d) in zip(zip(*got[0][1:]), zip(*got[1][1:])):
        if bits == 32:
            assert torch.equal(p, q) and torch.equal(c, d)
        else:
            assert ((p - q).abs() <= 3 * (2 * host.U * q.abs() + 2.0 ** -21 * 10 * host.HYPER["lr"])).all() and torch.equal(d, q.bfloat16())


@pytest.mark.parametrize("size,eps", [(1e6, 1e-8), (1e17, 1e-8), (1.0, 1e-12), (1e-18, 1e-30), (3e3, 0.0)])
def test_scales_and_eps_of_any_size(size, eps):
    """8-bit moments whose scales leave the range of the short way, or an eps that a subnormal root counts next to: the host's bits."""
    got = []
    for device in ("cpu", "cuda"):
        ps, gs, _, _ = host.tensors([3000, 5], (torch.float32, torch.float32), "cpu")
        gs = [g * size for g in gs]
        gs[0][1000:1512] /= size  # two blocks of ordinary size among them
        ps, gs = [p.to(device) for p in ps], [g.to(device) for g in gs]  # (the framework's division rounds by device)
        state = [ops.adamw_state8(p) for p in ps]
        ms, vs, ss = ([s[i] for s in state] for i in range(3))
        for t in (1, 2, 3):
            ops.adamw_step(ps, gs, ms, vs, step=t, lr=1e-2, eps=eps, scales=ss, seed=1)
        got.append(([x.cpu() for x in ms + vs + ss], [p.cpu() for p in ps]))
    # (blocks whose second moment is not finite have the scale NaN, and codes that say nothing)
    for k, (a, b) in enumerate(zip(got[0][0], got[1][0])):
        assert torch.equal(a.nan_to_num(-1.0), b.nan_to_num(-1.0)), k
    for p, q in zip(got[0][1], got[1][1]):
        assert torch.equal(p.isfinite(), q.isfinite())
        keep = p.isfinite()
        # three steps, each off by a rounding of the parameter and 2^-21 of an update of at most 10 lr
        assert ((p - q).abs()[keep] <= (3 * (2 * host.U * q.abs() + 2.0 ** -21 * 10 * 1e-2))[keep]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_on(bits):
    """A captured step with its number on the device, replayed, does what as many calls do; a number of the host is refused."""
    def make():
        ps, gs, ms, vs = host.tensors([1000, 3], (torch.float32, torch.float32), "cuda")
        more = {}
        if bits == 8:
            state = [ops.adamw_state8(p) for p in ps]
            ms, vs, ss = ([s[i] for s in state] for i in range(3))
            more = dict(scales=ss)
        return ps, gs, ms, vs, more
    ps, gs, ms, vs, more = make()
    for t in range(1, 5):
        ops.adamw_step(ps, gs, ms, vs, step=t, **host.HYPER, **more)
    qs, gs, mq, vq, more = make()
    number = torch.zeros(1, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        number.add_(1)
        ops.adamw_step(qs, gs, mq, vq, step=number, **host.HYPER, **more)
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ps + ms + vs, qs + mq + vq))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        number.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            ops.adamw_step(qs, gs, mq, vq, step=3, **host.HYPER, **more)


def test_given_stream():
    ps, gs, ms, vs = host.tensors([1 << 20], (torch.float32, torch.float32), "cuda")
    qs, _, mq, vq = host.tensors([1 << 20], (torch.float32, torch.float32), "cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    ops.adamw_step(ps, gs, ms, vs, step=1, stream=side, **host.HYPER)
    side.synchronize()
    ops.adamw_step(qs, gs, mq, vq, step=1, **host.HYPER)
    assert torch.equal(ps[0], qs[0]) and torch.equal(ms[0], mq[0])


def test_more_elements_than_32_bits_count():
    """The elements behind the 2^32nd of one tensor: bf16 parameters and gradients, 8-bit moments, against a step of those alone."""
    n = (1 << 32) + 1000
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-1500:] = torch.randn(1500, device="cuda").bfloat16()
    m, v, s = ops.adamw_state8(p)
    ops.adamw_step([p], [g], [m], [v], step=1, scales=[s], **host.HYPER)
    q, h = torch.zeros(1512, dtype=torch.bfloat16, device="cuda"), g[-1512:].clone()  # whole blocks: 1512 = 5 * 256 + 232, as n ends
    assert (n - 1512) % 256 == 0
    m2, v2, s2 = ops.adamw_state8(q)
    ops.adamw_step([q], [h], [m2], [v2], step=1, scales=[s2], **host.HYPER)
    assert torch.equal(p[-1512:], q) and torch.equal(s[:, -6:], s2) and not p[:-1512].any()


@pytest.mark.parametrize("dtypes", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
def test_codes_are_those_of_64_bits(dtypes):
    host.check_codes("cuda", dtypes, 6_000_001)
