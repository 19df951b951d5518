"""Attention over a cache of 4 bits where its weights are hard to hold: small ones beside values that f16 has no room for once they are weighted, and scales of any size."""
import math

import pytest

torch = pytest.importorskip("torch")
from test_gpu_attention4 import check, forward  # noqa: E402
from test_gpu_kv4 import Cache4, backend, quantised  # noqa: E402, F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_heads,d,group,page,kind", [
    (4, 64, 32, 16, "f16"), (8, 128, 64, 32, "bf16"), (5, 80, 32, 16, "f16"), (4, 128, 64, 24, "bf16"), (2, 128, 32, 16, "bf16"), (16, 128, 32, 16, "f16"), (12, 192, 64, 16, "bf16"), (3, 256, 32, 40, "f16")])
def test_small_weights_beside_large_values(backend, q_heads, d, group, page, kind):  # noqa: F811
    """One key far above 30 000 equal ones, 22.3 bits of weight above each: these make 0.6 % of a row, and where their values are all of one sign, all of an output whose value the one
    key's token has at zero.  That token's other values have scales of 2000.  300 sequences share the pages, so a CTA has one of them, and a warp that meets the token an eighth of its
    tokens: were they lost, the output would be off by that eighth."""
    n = 30000
    one = Cache4([(1, n)], q_heads, 1, d, kind, page, group)
    one.q.fill_(1.0)
    x = torch.zeros((n, 1, d), dtype=torch.float64, device="cuda")
    x[3] = 22.3 * math.log(2.0) / math.sqrt(d)
    one.put(True, one.places(0), *quantised(x, group))
    x = torch.randn((n, 1, d), device="cuda", generator=one.gen).double()
    half = d // 2 // group * group
    x[..., half:] = x[..., half:] * 100.0 + 4000.0
    x[3, :, half:] = 0.0
    x[3, :, :half] = torch.linspace(-16000, 16000, half, device="cuda").double()
    one.put(False, one.places(0), *quantised(x, group))
    one.install(backend)
    seqs = 300
    table = one.table.expand(seqs, -1).contiguous()
    starts, lens = torch.arange(seqs + 1, dtype=torch.int32, device="cuda"), torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    q, out = one.q.expand(seqs, -1).contiguous(), torch.full((seqs, q_heads * d), 7.0, dtype=one.kind, device="cuda")
    batch = one.batch(page_table=table.data_ptr(), row_start=starts.data_ptr(), kv_len=lens.data_ptr(), n_seqs=seqs, n_rows=seqs)
    backend.attention_forward_device(0, batch, q.data_ptr(), out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
    for i in range(0, seqs, 29):
        check(one, out[i:i + 1])
    # and by one sequence's parts
    forward(backend, one)
    check(one)


@pytest.mark.parametrize("q_heads,d,group,page,kind", [
    (4, 64, 32, 16, "f16"), (8, 64, 64, 5, "bf16"), (8, 96, 32, 16, "bf16"), (5, 80, 64, 24, "f16"), (8, 128, 64, 16, "f16"), (16, 128, 32, 24, "f16"), (9, 192, 32, 16, "bf16"), (8, 256, 64, 16, "f16"),
    (16, 256, 32, 48, "bf16")])
def test_scales_of_every_size(backend, q_heads, d, group, page, kind):  # noqa: F811
    """Every token's values of a size of its own, 2^-4 to 2^15, so that scales lie on both sides of 4 and 256, and at them."""
    for lens in ([(1, 700), (1, 40), (1, 5000)], [(2, 900), (1, 1), (1, 65)]):
        c = Cache4(lens, q_heads, 1, d, kind, page, group)
        for i, (_, k) in enumerate(lens):
            c.put(True, c.places(i), *quantised(torch.randn((k, 1, d), device="cuda", generator=c.gen).double(), group))
            size = 2.0 ** torch.randint(-4, 16, (k, 1, 1), device="cuda", generator=c.gen).double()
            x = (torch.rand((k, 1, d), device="cuda", generator=c.gen).double() * 2 - 1) * size
            x[::3, :, ::group] = 0.0  # scales of exactly 4, 256 and next to them
            x[::3, :, 1::group] = (torch.tensor([3.998, 4.0, 4.004, 255.9, 256.0, 256.25], device="cuda").double() * 15).repeat(k)[:x[::3].shape[0], None, None]
            x[::3] = x[::3].clamp(min=0.0).minimum(x[::3, :, 1:2])
            c.put(False, c.places(i), *quantised(x, group))
        c.install(backend)
        forward(backend, c)
        backend.stream_check(0, torch.cuda.current_stream().cuda_stream)
        check(c)
