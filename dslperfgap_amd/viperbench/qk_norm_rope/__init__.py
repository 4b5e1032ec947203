"""qk_norm_rope: HIP backend (hip_impl)."""
