"""BERT masked-LM federated session over rows that hold several documents:
a separator token ends each, attention stays within it and falls off with
distance, and AdamW holds its states in 8 bits.  Small CPU version; on MI355X
attention, norms and the optimizer step run as HIP kernels.
"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from colearn_federated_learning_amd import driver_config, run

cfg = driver_config(4).override(
    rounds=2, num_clients=2, data__samples_per_client=8,
    data__seq_len=48, data__vocab_size=128, train__batch_size=4,
    train__dtype="float32", train__optimizer="adamw8",
    train__weight_decay=0.01, model__hidden_size=64, model__num_layers=2,
    model__num_heads=4, model__intermediate_size=128,
    model__doc_sep_token=100, model__attn_distance_bias=True,
    model__attn_dropout=0.0, model__fused_add_norm=True,
)
history = run(cfg)
for rec in history:
    print(f"round {rec['round']}: mlm_loss={rec['mean_client_loss']:.4f}")
