"""The cache is sized by the memory that is free once the weights are in 8 bits, without what the checkpoint's took on the way."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("folder", [False, True])
def test_the_cache_gets_what_the_weights_left(folder, monkeypatch, tmp_path):
    from llmserve import EngineConfig
    from llmserve.engine import runner as module
    from llmserve.weights import write_random_model

    # 0.4 GB of layers in bfloat16, 0.2 in 8 bits, 16 MB of embedding and head
    config = dict(architectures=["LlamaForCausalLM"], model_type="llama", vocab_size=2048, hidden_size=2048, intermediate_size=5632, num_hidden_layers=4,
                  num_attention_heads=16, num_key_value_heads=4, max_position_embeddings=256, rope_theta=10000.0, rms_norm_eps=1e-5,
                  tie_word_embeddings=False)
    per_layer = 2048 * (16 + 2 * 4) * 128 + 2048 * 2048 + 3 * 2048 * 5632
    seen = {}
    real = module.pool_sizes_for_budget

    def sized(groups, block_size, elem, budget, *rest):
        seen["budget"], seen["allocated"] = budget, torch.cuda.memory_allocated(DEV)
        torch.cuda.empty_cache()
        seen["free"] = torch.cuda.mem_get_info(torch.device(DEV))[0]
        return real(groups, block_size, elem, 64 << 20, *rest)

    monkeypatch.setattr(module, "pool_sizes_for_budget", sized)
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated(DEV)
    engine = EngineConfig(weights="float8", gpu_memory_fraction=0.5, max_num_seqs=2)
    if folder:
        write_random_model(tmp_path, config, seed=1)
        module.ModelRunner.from_folder(tmp_path, engine, DEV)
    else:
        module.ModelRunner.from_random(config, 1, engine, DEV)
    held = 4 * per_layer * 1.01 + 2 * 2048 * 2048 * 2 + (32 << 20)  # (scales, norms, tables: some)
    assert seen["allocated"] - before <= held
    assert seen["budget"] >= 0.5 * (seen["free"] - (32 << 20))
