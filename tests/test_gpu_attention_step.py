"""GPU: the operators of an attention layer one behind the other, as a model step runs them: index
preparation, head norm + rotary embedding + cache write, attention over the pages - and the same
batch with its common prefix read once - against the 64-bit formulas."""
import copy

import pytest
import torch

import workloads as W
from lmserve_b200.model_step import ModelStepCache
from lmserve_b200.ops import paged_attention, qk_norm_rotary_pos_emb_and_cache, shared_prefix_attention
from lmserve_b200.step_inputs import InferInput
from oracle import attention_oracle, rope_oracle, step_oracle
from test_paged_attention import compare

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def layer_inputs(T, HQ, H, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (HQ + 2 * H) * D, generator=g).to(dtype)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2))
    cuts = (slice(0, HQ * D), slice(HQ * D, (HQ + H) * D), slice((HQ + H) * D, None))
    return [qkv[:, c] for c in cuts] + [qw, kw], [qkv.to(DEV)[:, c] for c in cuts] + [qw.to(DEV), kw.to(DEV)]


@pytest.mark.parametrize("dtype,HQ,H,D", [(torch.bfloat16, 8, 2, 128), (torch.float16, 14, 2, 64)])
def test_model_steps(dtype, HQ, H, D):
    L, NB, BS = 2, 200, 16
    kv = torch.randn(L, NB, 2, BS, H, D, device=DEV).to(dtype)
    step_cache = ModelStepCache(kv, stream=torch.cuda.Stream(), max_batch=32, max_tokens=1024, max_blocks=512)
    table = rope_oracle.build_cos_sin_cache(2048, D, dtype)
    on_gpu = table.to(DEV)
    for step in range(3):
        reqs = W.make_step_requests(NB, BS, [6, 0, 5][step], 1, 200, [3, 2, 0][step], 20, 150, seed=40 + step)
        ref = step_oracle.make_inputs(copy.deepcopy(reqs), BS)
        _, params = step_cache.begin_step(reqs)
        T = params.position_ids.shape[0]
        with torch.cuda.stream(step_cache.stream):
            for layer in range(L):
                (q, k, v, qw, kw), d = layer_inputs(T, HQ, H, D, dtype, 100 * step + layer)
                rotated = qk_norm_rotary_pos_emb_and_cache(*d, params.position_ids, on_gpu, D, kv[layer], params.slot_mapping)
                out = step_cache.attend_layer(layer, rotated, params)
                step_cache.stream.synchronize()
                # the rows written
                positions = torch.from_numpy(ref["position_ids"]).long()
                exact, bound = attention_oracle.qk_norm_rotary(k, kw, positions, table, D, 1e-6)
                slots = torch.from_numpy(ref["slot_mapping"]).long()
                cache = kv[layer].cpu()
                written = cache[slots // BS, :, slots % BS]
                assert ((written[:, 0].reshape(T, -1).double() - exact).abs() <= bound).all()
                assert torch.equal(written[:, 1].reshape(T, -1).view(torch.int16), v.contiguous().view(torch.int16))
                # the attention over them (both phases of the batch as one list of requests)
                own = tuple(torch.from_numpy(ref[n]) for n in ("kv_block_indptrs", "kv_block_indices", "kv_last_block_lens"))
                want = attention_oracle.paged_attention(rotated.cpu().view(T, HQ, D), cache[:, 0], cache[:, 1], own,
                                                        torch.from_numpy(ref["cu_seqlens_q"]))
                o, ob = want[:2]
                assert ((out.cpu().double().view(T, HQ, D) - o).abs() <= ob).all()


def test_a_batch_behind_a_common_prompt():
    """Four requests decode behind the same three full blocks: one table each, or the blocks once."""
    dtype, HQ, H, D, BS, NB = torch.bfloat16, 8, 2, 128, 16, 64
    kv = torch.randn(1, NB, 2, BS, H, D, device=DEV).to(dtype)
    step_cache = ModelStepCache(kv, max_batch=8, max_tokens=64, max_blocks=128)
    shared = [60, 3, 41]
    reqs = []
    for i, n in enumerate((5, 30, 16, 1)):      # own tokens, the new one included
        blocks = shared + list(range(5 + 4 * i, 5 + 4 * i + -(-n // BS)))
        reqs.append(InferInput(input_ids=[7], input_len=1, filled_token_len=48 + n - 1, context_len=48 + n, block_ids=blocks))
    _, params = step_cache.begin_step(reqs)
    (q, k, v, qw, kw), d = layer_inputs(4, HQ, H, D, dtype, 9)
    table = rope_oracle.build_cos_sin_cache(256, D, dtype).to(DEV)
    rotated = qk_norm_rotary_pos_emb_and_cache(*d, params.position_ids, table, D, kv[0], params.slot_mapping)
    whole = step_cache.attend_layer(0, rotated, params)
    x = params.decode
    alone, lse = paged_attention(rotated, kv[0], x.kv_indptr, x.kv_indices, x.kv_last_page_len, return_lse=True)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    counts = [len(r.block_ids) - 3 for r in reqs]
    own = (i32([0] + list(torch.tensor(counts).cumsum(0))), i32(sum((list(r.block_ids[3:]) for r in reqs), [])), x.kv_last_page_len)
    prefix = (i32([0, 3]), i32(shared), i32([BS]))
    split, split_lse = shared_prefix_attention(rotated, kv[0], *prefix, *own, return_lse=True)
    cache = kv[0].cpu()
    cpu = lambda t: tuple(a.cpu() for a in t)
    want = attention_oracle.paged_attention(rotated.cpu().view(4, HQ, D), cache[:, 0], cache[:, 1], cpu(own), prefix=cpu(prefix))
    compare(split, split_lse, want)
    compare(alone, lse, want)
    assert torch.equal(whole.view(torch.int16), alone.view(torch.int16))
