"""Arguments that attention_kv8 refuses, beside those of test_gpu_kv_attention."""
import pytest
import torch
from test_gpu_kv_attention import i32

pytestmark = pytest.mark.gpu


def call(jkb, q, out, lse=None, starts=(0, 3)):
    cache = jkb.KvCache(2, 16, 1, q.shape[2])
    jkb.attention_kv8(out, q, cache, jkb.AttentionWorkspace(cache), i32([[0]]), i32([3]),
                      i32(starts), 3, 0.1, lse=lse)


def test_lse_of_another_shape(jkb):
    """[heads, tokens] or flat memory would be filled as [tokens, heads]."""
    q = torch.zeros(3, 4, 64, device="cuda")
    out = torch.empty_like(q)
    call(jkb, q, out, torch.empty(3, 4, device="cuda"))
    for lse in (torch.empty(4, 3, device="cuda"), torch.empty(12, device="cuda"),
                torch.empty(3, 4, 1, device="cuda"), torch.empty(4, 3, device="cuda").T):
        with pytest.raises(ValueError):
            call(jkb, q, out, lse)
    q = q[:0]
    call(jkb, q, out[:0], torch.empty(0, 4, device="cuda"), (0, 0))


@pytest.mark.parametrize("heads", [1, 3])
def test_more_query_rows_than_row_numbers(jkb, heads):
    """Broadcast rows, of which there is one in memory: refused before anything runs."""
    n = 2**31 // heads - 100 // heads
    q = torch.zeros(1, heads, 8, device="cuda").expand(n, heads, 8)
    with pytest.raises(jkb.TensorBoundsError):
        call(jkb, q, torch.zeros(1, heads, 8, device="cuda").expand(n, heads, 8), starts=(0, n))
