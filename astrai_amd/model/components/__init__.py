from astrai_amd.model.components import int8, mlp, scored_moe  # noqa: F401  (registers the FFN components)
