"""One draw per row at the vocabularies where the number of CTAs that hold a row changes."""
import pytest

from .test_sample_rows import draw, logits, us

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [c * 20040 + d for c in (1, 2, 4, 8) for d in (-7, 0, 1, 440)])
def test_draws_around_the_sizes_of_a_cluster(dtype, vocab):
    n = 160 if vocab < 41000 else 9
    x = logits(n, vocab, vocab, dtype)
    if n > 9:                                # (few rows take more CTAs: enough of them, few compared)
        from emberllm_b200 import sample_rows
        u = torch.tensor(us(n, vocab)).cuda()
        out = torch.full((n,), -1, dtype=torch.int32, device="cuda")
        sample_rows(x, out, u)
        some = torch.tensor([0, 1, 80, 147, 148, 159])
        assert out.cpu()[some].tolist() == draw(x[some.cuda()], us(n, vocab)[some.numpy()]).tolist()
    else:
        draw(x, us(n, vocab), top_p=0.9)
        draw(x, us(n, vocab), temperature=0.8, top_k=60, min_p=0.01)
