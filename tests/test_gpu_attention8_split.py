"""GPU: what a request gets from the 8-bit cache does not depend on what else is in the batch, by which its list is cut another way."""
import pytest
import torch

from tests._attention import attend as reference, check_out
from tests._cache8 import cache_of
from tests.test_gpu_attention import make
from tests.test_gpu_attention8 import F16, BF16
from valora_amd.attention import AttentionPlan

pytestmark = pytest.mark.gpu
FEW, TALL = 0, 1           # words of the plan: records of either list


def attend(dev, c, page, which):
    """The requests `which` of a case in a plan of their own: (rows of each, records of the plan's lists)."""
    hq, d, hkv = c["q"].shape[1], c["q"].shape[2], c["kb"].shape[1]
    i32 = lambda t: torch.tensor(t, dtype=torch.int32, device=dev)  # noqa: E731
    news = [c["news"][b] for b in which]
    starts = [sum(news[:i]) for i in range(len(which))]
    q = torch.cat([c["q"][c["starts"][b]:c["starts"][b] + c["news"][b]] for b in which]).to(dev)
    plan = AttentionPlan(i32(starts), i32(news), i32([c["lens"][b] for b in which]), n_tokens=sum(news), max_seq_len=max(news),
                         max_kv_len=max(c["lens"][b] for b in which), q_heads=hq, kv_heads=hkv, head_dim=d, page_size=page)
    args = [c[n].to(dev) for n in ("key_codes", "value_codes", "powers")] + [c["table"][list(which)].to(dev)]
    outs = []
    for _ in range(3):
        out = torch.full_like(q, 7.0)
        plan.attend8(out, q, *args)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs[1:])
    return outs[0].split(news), plan.buf.view(torch.int32)[[FEW, TALL]].tolist()


@pytest.mark.parametrize("dtype,hq,hkv,d,page", [(F16, 8, 2, 128, 2), (BF16, 4, 4, 64, 16), (BF16, 4, 2, 96, 2)])
def test_requests_alone_and_in_a_batch(dev, dtype, hq, hkv, d, page):
    """Decoding requests and chunks, alone in many pieces and among hundreds of others in few: all within the bound of the definition, which is the
    same."""
    some = [(1, 3000), (1, 40), (64, 900), (3, 2500), (150, 1500)]
    c = make(dev, dtype, hq, hkv, d, page, some + [(1, 150 + 7 * i % 70) for i in range(800)], seed=12)
    c["key_codes"], c["value_codes"], c["powers"], c["kb"], c["vb"] = cache_of(c["kb"], c["vb"], page, dtype)
    together, (few, tall) = attend(dev, c, page, range(len(c["news"])))
    cut_alone = 0
    for b, (n, length) in enumerate(some):
        alone, records = attend(dev, c, page, [b])
        cut_alone += sum(records)
        at = c["starts"][b]
        want, _, bound, _ = reference(c["q"][at:at + n], c["kb"], c["vb"], c["table"][b:b + 1], [0], [n], [length], page, 0, d ** -0.5)
        check_out(alone[0], want, bound)
        check_out(together[b], want, bound)
    # (the others' 800 records aside, the same requests are in fewer pieces)
    assert few + tall - 800 < cut_alone
