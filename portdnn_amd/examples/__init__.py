"""Programs that use the operators together."""
